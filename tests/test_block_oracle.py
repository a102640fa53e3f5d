"""The block operators' oracle on the CPU: its gradients against differences, its rotation against complex
multiplication, its layouts against the ones the packing function writes; and the checks of arguments that need no GPU."""
import itertools
import math
import os
import re

import pytest
import torch

from lingbot_world_v2_realtime_amd import _lib, kernels
from lingbot_world_v2_realtime_amd.layers.linear import W4Linear, convert_to_w4
from lingbot_world_v2_realtime_amd.layers.norm import gated_norm
from lingbot_world_v2_realtime_amd.layers.rotary import Rotary, grid_positions, rotary_embed
from oracle import block

HEADER = os.path.join(os.path.dirname(__file__), "..", "include", "lbw_block.h")
OK, E_NULL, E_SHAPE, E_ALIGN, E_DEVICE = range(5)
FAKE = 1 << 20   # a 16-byte aligned non-null address, never dereferenced on these paths


def _g(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("norm,post,mod", itertools.product([None, "layer", "rms"], [None, "layer", "rms"],
                                                             ["shared", "rows"]))
def test_norm_gradients_against_differences(norm, post, mod):
    """Central differences of the float64 oracle's own outputs, with a step of 1e-5: the error of a difference is about
    step^2 times a third derivative (1e-10 times O(100)) plus 1e-16 / 1e-5."""
    g = _g(3)
    b, n, c = 2, 5, 6
    shape = (c,) if mod == "shared" else (b, 2, c)
    a = {"x": torch.randn(b, n, c, generator=g), "y": torch.randn(b, n, c, generator=g),
         "gate": torch.randn(shape, generator=g), "post_weight": torch.randn(c, generator=g)}
    if norm is not None:
        a |= {"shift": torch.randn(shape, generator=g), "scale": torch.randn(shape, generator=g),
              "weight": torch.randn(c, generator=g), "bias": torch.randn(c, generator=g)}
    a = {k: v.double() for k, v in a.items()}
    kw = dict(norm=norm, post_norm=post, residual_scale=0.8, branch_scale=1.3)
    ds = torch.randn(b, n, c, generator=g).double()
    dh = torch.randn(b, n, c, generator=g).double() if norm is not None else None

    def total(t):
        (s, _), (h, _), _ = block.gated_norm(**t, **kw)
        return float((s * ds).sum() + ((h * dh).sum() if dh is not None else 0))

    grads = block.gated_norm(**a, **kw, ds=ds, dh=dh)[2]
    assert set(grads) == set(a)
    for name, v in a.items():
        for at in range(0, v.numel(), 3):
            lo, hi = v.clone(), v.clone()
            lo.view(-1)[at] -= 1e-5
            hi.view(-1)[at] += 1e-5
            want = (total({**a, name: hi}) - total({**a, name: lo})) / 2e-5
            assert abs(float(grads[name][0].reshape(-1)[at]) - want) < 1e-6 * (1 + abs(want)), name


def test_rotary_against_complex_numbers():
    g = _g(4)
    x = torch.randn(2, 3, 2, 10, generator=g).double()
    pos = torch.tensor([[0, 5, 1 << 20], [7, 8, 9]])
    freq = torch.tensor([1.0, 0.1, 1e-3], dtype=torch.float64)
    for pairs in ("interleaved", "half"):
        out, _ = block.rotary(x, pos, freq, pairs=pairs, factor=1.5)
        z = torch.complex(x[..., 0:6:2], x[..., 1:6:2]) if pairs == "interleaved" else \
            torch.complex(x[..., :3], x[..., 3:6])
        z = z * 1.5 * torch.exp(1j * (pos[..., None] * freq))[:, :, None]
        got = torch.complex(out[..., 0:6:2], out[..., 1:6:2]) if pairs == "interleaved" else \
            torch.complex(out[..., :3], out[..., 3:6])
        assert torch.allclose(got, z, rtol=0, atol=1e-12) and torch.equal(out[..., 6:], x[..., 6:])
        back, _ = block.rotary(out, pos, freq, pairs=pairs, factor=1 / 1.5, inverse=True)
        assert torch.allclose(back, x, rtol=0, atol=1e-12)


def test_rotary_plans():
    """The stretched frequencies: ends of every rule, and one section's table equal to the model's."""
    from lingbot_world_v2_realtime_amd.layers.prologue import rope_freqs
    plain = Rotary.build(64, "cpu")
    assert torch.equal(Rotary.build(64, "cpu", scaling="linear", stretch=4.0).freq, plain.freq / 4)
    base = Rotary.build(64, "cpu", scaling="base", stretch=4.0).freq
    assert base[0] == plain.freq[0] and math.isclose(base[-1], plain.freq[-1] / 4, rel_tol=1e-12)
    ramp = Rotary.build(64, "cpu", scaling="ramp", stretch=4.0, trained_len=2048)
    turns = 2048 * plain.freq / (2 * math.pi)
    assert torch.equal(ramp.freq[turns >= 32], plain.freq[turns >= 32])
    assert torch.allclose(ramp.freq[turns <= 1], plain.freq[turns <= 1] / 4, rtol=1e-15)
    assert bool((ramp.freq[:-1] > ramp.freq[1:]).all()) and math.isclose(ramp.factor, 1 + 0.1 * math.log(4))
    three = Rotary.build(128, "cpu", sections=(22, 21, 21))
    assert three.axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    table = rope_freqs("cpu")   # row 1: the angles of position 1, so cos of the frequencies
    assert torch.allclose(three.freq.cos(), table[1, :, 0], rtol=0, atol=1e-14)
    pos = grid_positions((2, 3, 4), 5, "cpu")
    assert pos.shape == (24, 3) and pos[0].tolist() == [5, 0, 0] and pos[23].tolist() == [6, 2, 3]
    for bad in (dict(dim=63), dict(dim=64, sections=(30, 1)), dict(dim=64, sections=(32, 0)), dict(dim=64, stretch=0.5),
                dict(dim=64, scaling="other"), dict(dim=64, scaling="ramp", stretch=2.0)):
        with pytest.raises(ValueError):
            Rotary.build(**bad, device="cpu")


@pytest.mark.parametrize("fmt,zeros,group", [("int4", False, 128), ("int4", True, 32), ("fp4", False, 64)])
def test_pack_w4_layout(fmt, zeros, group):
    """pack_w4's tiles, read back word by word from the layout's definition."""
    g = _g(5)
    n, k = 37, 300
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scale = torch.rand(n, groups, generator=g).to(torch.bfloat16)
    zero = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    w4, sc, z = kernels.pack_w4(codes, scale, zero, fmt)
    assert w4.shape == (3, 3, 1024) and sc.shape == (3, 3, 16, 128 // group)
    full = block.unpack_w4(w4, fmt)
    assert torch.equal(full[:n, :k], codes) and not full[n:].any() and not full[:, k:].any()
    assert torch.equal(block.unpack_scale(sc)[:n, :groups], scale) and not block.unpack_scale(sc)[n:].any()
    assert (z is None) if zero is None else torch.equal(block.unpack_scale(z)[:n, :groups], zero)


def test_quant_w4_oracle_is_within_half_a_step():
    g = _g(6)
    w = torch.randn(8, 256, generator=g)
    for fmt, zeros in (("int4", False), ("int4", True), ("fp4", False)):
        codes, scale, zero = block.quant_w4(w, 64, fmt, zeros)
        v = block.w4_values(codes, scale, zero, fmt)
        step = scale.float().repeat_interleave(64, 1)
        # integer codes: half a step (and up to another half where a rounded scale or zero ends the range early);
        # fp4: half of the widest gap, 2 steps
        assert bool(((v - w).abs() <= step * (1.0 if fmt == "fp4" else 1.01) + 0.05 * step).all())


# ---------------------------------------------------------------- refusals


def test_block_header_declarations_are_bound_and_exported():
    src = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    decl = {m.group(1): m.group(2).count(",") + 1
            for m in re.finditer(r"^\s*\w+\s+(lbw_\w+)\s*\(([^)]*)\)\s*;", src, flags=re.M)}
    assert set(decl) == set(_lib.BLOCK_SIGNATURES) and len(decl) == 6
    lib = _lib.load()
    for name, n in decl.items():
        assert len(_lib.BLOCK_SIGNATURES[name][1]) == n and hasattr(lib, name), name
    assert f"#define LBW_NORM_MAX_WIDTH {kernels.NORM_MAX_WIDTH}" in src
    assert f"#define LBW_ROTARY_MAX_DIM {kernels.ROTARY_MAX_DIM}" in src


def _norm(**kw):
    a = dict(x=FAKE, y=FAKE, dtype=0, vec=2, batch=1, len=10, width=64, xs=(640, 64), ys=(640, 64), gate=(None, 0, 0),
             shift=(None, 0, 0), scale=(None, 0, 0), group_len=10, weight=None, bias=None, post_weight=None, norm=1,
             post=0, s=FAKE, h=FAKE)
    a.update(kw)
    return _lib.load().lbw_gated_norm(
        a["x"], a["y"], a["dtype"], a["vec"], a["batch"], a["len"], a["width"], *a["xs"], *a["ys"], *a["gate"],
        *a["shift"], *a["scale"], a["group_len"], a["weight"], a["bias"], a["post_weight"], a["norm"], a["post"],
        1e-6, 1.0, 1.0, a["s"], a["h"], None)


def _norm_bwd(**kw):
    a = dict(ds=FAKE, dh=FAKE, x=FAKE, y=FAKE, dtype=0, vec=2, batch=1, len=10, width=64, gate=(FAKE, 64, 64),
             scale=(FAKE, 64, 64), rowwise=7, groups=1, group_len=10, weight=FAKE, bias=FAKE, post_weight=None, norm=1,
             post=0, dx=FAKE, dy=FAKE, dgate=None, dshift=None, dscale=None, dweight=None, dbias=None,
             dpost_weight=None, ws=FAKE)
    a.update(kw)
    return _lib.load().lbw_gated_norm_bwd(
        a["ds"], a["dh"], a["x"], a["y"], a["dtype"], a["vec"], a["batch"], a["len"], a["width"], 640, 64, 640, 64,
        *a["gate"], *a["scale"], a["rowwise"], a["groups"], a["group_len"], a["weight"], a["bias"], a["post_weight"],
        a["norm"], a["post"], 1e-6, 1.0, 1.0, a["dx"], a["dy"], a["dgate"], a["dshift"], a["dscale"], a["dweight"],
        a["dbias"], a["dpost_weight"], a["ws"], None)


def test_gated_norm_entry_point_refusals():
    assert _norm(x=None) == E_NULL
    assert _norm(h=None) == E_NULL
    assert _norm(norm=0, h=None, s=None) == E_NULL
    assert _norm(norm=0) == E_NULL                                     # an output that nothing would write
    assert _norm(y=None, gate=(FAKE, 0, 0)) == E_NULL
    assert _norm(y=None, post=1) == E_NULL
    assert _norm(dtype=3) == E_SHAPE and _norm(dtype=-1) == E_SHAPE
    assert _norm(dtype=0, vec=1) == E_SHAPE
    assert _norm(width=0) == E_SHAPE and _norm(width=12289) == E_SHAPE
    assert _norm(len=0) == E_SHAPE and _norm(batch=1 << 20, len=1 << 20) == E_SHAPE
    assert _norm(batch=1 << 62, len=1 << 62) == E_SHAPE
    assert _norm(group_len=0) == E_SHAPE
    assert _norm(norm=3) == E_SHAPE and _norm(post=-1) == E_SHAPE
    assert _norm(norm=0, h=None, weight=FAKE) == E_SHAPE
    assert _norm(x=FAKE + 1) == E_ALIGN and _norm(gate=(FAKE + 2, 0, 0)) == E_ALIGN
    assert _norm_bwd(ds=None, dh=None) == E_NULL
    assert _norm_bwd(dgate=FAKE, ws=None) == E_NULL
    assert _norm_bwd(dgate=FAKE, gate=(None, 0, 0)) == E_NULL
    assert _norm_bwd(dh=None, dshift=FAKE) == E_NULL
    assert _norm_bwd(dpost_weight=FAKE) == E_NULL
    assert _norm_bwd(groups=2, group_len=4) == E_SHAPE                # tokens 8, 9 have no row
    assert _norm_bwd(groups=0) == E_SHAPE
    assert _norm_bwd(batch=1 << 30, len=1, width=4096, dgate=FAKE) == E_SHAPE   # more workgroups than a grid has
    assert _norm_bwd(dgate=FAKE, ws=FAKE + 8) == E_ALIGN
    lib = _lib.load()
    assert lib.lbw_gated_norm_bwd_workspace_bytes(0, 1, 64, 1, 1) == 0
    assert lib.lbw_gated_norm_bwd_workspace_bytes(1, 100, 64, 1, 100) % (3 * 64 * 4) == 0


def _rotary(**kw):
    a = dict(q=FAKE, k=FAKE, dtype=0, batch=1, len=4, qh=2, kh=1, dim=64, pairs=32, pos=None, freq=FAKE, axis=None,
             axes=1, qo=FAKE, ko=FAKE)
    a.update(kw)
    return _lib.load().lbw_rotary(a["q"], a["k"], a["dtype"], a["batch"], a["len"], a["qh"], a["kh"], a["dim"],
                                  a["pairs"], 512, 128, 64, 256, 64, 64, a["pos"], 1, 4, 1, 0, 0, a["freq"], a["axis"],
                                  a["axes"], 1, 0, 1.0, a["qo"], a["ko"], 512, 128, 64, 256, 64, 64, None)


def test_rotary_entry_point_refusals():
    assert _rotary(q=None) == E_NULL and _rotary(ko=None) == E_NULL and _rotary(freq=None) == E_NULL
    assert _rotary(dtype=3) == E_SHAPE and _rotary(len=0) == E_SHAPE and _rotary(qh=0) == E_SHAPE
    assert _rotary(dim=32) == E_SHAPE and _rotary(pairs=0) == E_SHAPE and _rotary(dim=514) == E_SHAPE
    assert _rotary(axes=0) == E_SHAPE and _rotary(batch=1 << 61, len=1 << 61) == E_SHAPE
    assert _rotary(q=FAKE + 1) == E_ALIGN and _rotary(freq=FAKE + 4) == E_ALIGN and _rotary(pos=FAKE + 4) == E_ALIGN


def _gemm(**kw):
    a = dict(x=FAKE, dtype=0, m=3, k=100, xs=100, w4=FAKE, scale=FAKE, zero=None, fmt=0, group=64, n=30, bias=None,
             out=FAKE)
    a.update(kw)
    return _lib.load().lbw_gemm_w4(a["x"], a["dtype"], a["m"], a["k"], a["xs"], a["w4"], a["scale"], a["zero"],
                                   a["fmt"], a["group"], a["n"], a["bias"], a["out"], None)


def test_w4_entry_point_refusals():
    assert _gemm(x=None) == E_NULL and _gemm(w4=None) == E_NULL and _gemm(scale=None) == E_NULL and _gemm(out=None) == E_NULL
    assert _gemm(dtype=2) == E_SHAPE and _gemm(m=0) == E_SHAPE and _gemm(m=(1 << 24) + 1) == E_SHAPE
    assert _gemm(k=0) == E_SHAPE and _gemm(n=0) == E_SHAPE and _gemm(group=16) == E_SHAPE and _gemm(fmt=2) == E_SHAPE
    assert _gemm(fmt=1, zero=FAKE) == E_SHAPE
    assert _gemm(x=FAKE + 1) == E_ALIGN and _gemm(w4=FAKE + 8) == E_ALIGN and _gemm(scale=FAKE + 1) == E_ALIGN
    q = _lib.load().lbw_quant_w4
    assert q(None, 0, 8, 8, 8, 0, 64, FAKE, FAKE, None, None) == E_NULL
    assert q(FAKE, 0, 8, 8, 8, 1, 64, FAKE, FAKE, FAKE, None) == E_SHAPE
    assert q(FAKE, 0, 8, 0, 8, 0, 64, FAKE, FAKE, None, None) == E_SHAPE
    assert q(FAKE, 0, (1 << 20), 8, 8, 0, 64, FAKE, FAKE, None, None) == E_SHAPE
    assert q(FAKE + 2, 1, 8, 8, 8, 0, 64, FAKE, FAKE, None, None) == E_ALIGN


def test_host_tensors_are_refused():
    x = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        gated_norm(x)
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        rotary_embed(q, None, 0, Rotary.build(64, "cpu"))
    with pytest.raises(ValueError, match="device tensor"):
        kernels.quant_w4(torch.zeros(8, 8))
    with pytest.raises(ValueError, match="device tensor"):
        kernels.gemm_w4(torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(1, 1, 1024, dtype=torch.uint8),
                        torch.zeros(1, 1, 16, 1, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        gated_norm(x.double())
    with pytest.raises(TypeError):
        kernels.gemm_w4(torch.zeros(2, 128), None, None)


def test_lazy_and_learned_arguments_are_refused():
    """A negation that is not in memory yet, and a factor given as a tensor, whose gradient a number would lose."""
    x = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="negated"):
        gated_norm(torch._neg_view(x))
    with pytest.raises(ValueError, match="negated"):
        rotary_embed(torch._neg_view(x.view(1, 4, 1, 64)), None, 0, Rotary.build(64, "cpu"))


def test_pack_w4_refusals():
    codes, scale = torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4, 1)
    for bad in (dict(codes=codes.int()), dict(codes=codes[0]), dict(scale=torch.ones(4, 3)), dict(scale=torch.ones(3, 1)),
                dict(fmt="int8"), dict(fmt="fp4", zero=torch.zeros(4, 1)), dict(zero=torch.zeros(4, 2))):
        with pytest.raises(ValueError):
            kernels.pack_w4(**{"codes": codes, "scale": scale, **bad})


def test_convert_to_w4_selects(monkeypatch):
    """Which linears are replaced; the quantisation itself needs the GPU."""
    monkeypatch.setattr(kernels, "quant_w4", lambda w, group, fmt, zeros: (
        torch.zeros(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.bfloat16), None))
    net = torch.nn.Sequential(torch.nn.Linear(1024, 1536), torch.nn.Linear(1536, 512), torch.nn.GELU())
    assert convert_to_w4(net) == (1, 2)
    assert isinstance(net[0], W4Linear) and type(net[1]) is torch.nn.Linear and net[0].out_features == 1536


def test_convert_to_w4_shared_and_derived(monkeypatch):
    """A linear that stands in two places is replaced in both by one module; a subclass (its owner may read its weight, as
    nn.MultiheadAttention does) stays."""
    monkeypatch.setattr(kernels, "quant_w4", lambda w, group, fmt, zeros: (
        torch.zeros(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.bfloat16), None))
    lin = torch.nn.Linear(1024, 1024)
    net = torch.nn.ModuleDict({"a": torch.nn.Sequential(lin, torch.nn.GELU(), lin), "b": torch.nn.MultiheadAttention(1024, 8)})
    assert convert_to_w4(net) == (1, 1)
    assert isinstance(net["a"][0], W4Linear) and net["a"][2] is net["a"][0]
    assert isinstance(net["b"].out_proj, torch.nn.Linear)
