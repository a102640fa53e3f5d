"""The block operators on the GPU against their definitions in 64 bits (oracle/block.py).

Every bound is half a step of the output's type plus K * 2^-24 times the magnitude of what was added and multiplied on the
way (the oracle's second value): K counts the 32-bit roundings on the longest path. Norms: a thread adds at most 24 values of a row in
turn and the team 6 + 8 partial sums, twice for a variance, with a few products around: K = 96. Sums over rows: at most
rows / 8 in a thread's turn and 8 + chunks / 16 + 16 + modulation rows / 16 after that, under 160 for the sizes here, on
terms with the norm's own errors: K = 256. Rotations: two products, a sum, and a sine whose reduced angle is rounded to 2^-25 of
a half turn (3.2 * 2^-24 in radians) and whose last bits are good to 4 * 2^-24: K = 12.
4-bit products: one rounding for 32 columns, one for a group and for a wave: K = columns / 16 + 24.
"""
import itertools

import pytest
import torch

from oracle import block

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS32 = 2.0 ** -24


def _within(got, want, what, k):
    value, mag = want
    assert got.shape == value.shape, what
    half = torch.finfo(got.dtype).eps / 2
    # (the smallest numbers of fp16 are a fixed step apart)
    tol = half * (value.abs() + k * EPS32 * mag) + k * EPS32 * mag + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - value).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of its bound (max error {err.max().item():.3e})"


def _rand(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _norm_inputs(seed, b, n, c, dtype="bf16", vec=None, norm="layer", post=None, mod="rows", rows=3, affine=True):
    g = _rand(seed)

    def new(*shape, std=1.0, mean=0.0, dt=DT[dtype]):
        return (torch.randn(*shape, device=DEV, generator=g) * std + mean).to(dt)

    v = DT[vec or dtype]
    a = {"x": new(b, n, c, std=2.0, mean=0.3), "y": new(b, n, c)}
    shape = {"none": None, "shared": (c,), "rows": (b, rows, c)}[mod]
    if shape is not None:
        a["gate"] = new(*shape, dt=v)
        if norm is not None:
            a["shift"], a["scale"] = new(*shape, std=0.5, dt=v), new(*shape, std=0.5, dt=v)
    if affine:
        a["post_weight"] = new(c, std=0.3, mean=1.0, dt=v)
        if norm is not None:
            a["weight"], a["bias"] = new(c, std=0.3, mean=1.0, dt=v), new(c, std=0.3, dt=v)
    return a


def _check_norm(a, what, ds=None, dh=None, **kw):
    from lingbot_world_v2_realtime_amd import gated_norm, kernels
    a = {k: v.detach().requires_grad_() for k, v in a.items()}
    out = gated_norm(**a, **kw)
    with torch.no_grad():
        again = gated_norm(**a, **kw)
    s, h, grads = block.gated_norm(**a, **kw, ds=ds, dh=dh)
    has_s, has_h = "y" in a, kw.get("norm", "layer") is not None
    want = [w for w, has in ((s, has_s), (h, has_h)) if has]
    out, again = ((o,) if isinstance(o, torch.Tensor) else o for o in (out, again))
    assert len(out) == len(want)
    for o, o2, w in zip(out, again, want):
        assert o.dtype == a["x"].dtype and o.is_contiguous() and torch.equal(o, o2)
        _within(o.detach(), w, f"{what}: output", 96)
    if ds is None and dh is None:
        return
    names = list(a)
    d = [x for x, has in ((ds, has_s), (dh, has_h)) if has]
    kept = [(o, x) for o, x in zip(out, d) if x is not None]
    got = torch.autograd.grad([o for o, _ in kept], list(a.values()), [x for _, x in kept], allow_unused=True)
    del kernels
    for name, gr in zip(names, got):
        if gr is None:
            assert not grads[name][0].any(), name
            continue
        assert gr.dtype == a[name].dtype
        _within(gr, grads[name], f"{what}: d_{name}", 96 if name in ("x", "y") else 256)


NORM_SIZES = [(1, 1, 8), (1, 1, 1), (2, 5, 7), (1, 33, 1536), (3, 70, 771), (1, 9, 5120), (2, 3, 8192), (1, 2, 12288),
              (2, 19, 2056), (1, 300, 256), (1, 4, 12285)]


@pytest.mark.parametrize("b,n,c", NORM_SIZES)
@pytest.mark.parametrize("dtype,vec", [("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_gated_norm_sizes(b, n, c, dtype, vec):
    a = _norm_inputs(b * n + c, b, n, c, dtype, vec, rows=min(3, n))
    g = _rand(7)
    ds, dh = (torch.randn(b, n, c, device=DEV, generator=g).to(DT[dtype]) for _ in range(2))
    _check_norm(a, f"{b}x{n}x{c} {dtype}/{vec}", ds, dh, norm="layer")


@pytest.mark.parametrize("norm,post,mod,affine", itertools.product([None, "layer", "rms"], [None, "layer", "rms"],
                                                                   ["none", "shared", "rows"], [False, True]))
def test_gated_norm_forms(norm, post, mod, affine):
    if norm is None and post is None and mod == "none" and not affine:
        pass   # a plain scaled addition: still a call
    a = _norm_inputs(11, 2, 41, 520, "bf16", "bf16", norm, post, mod, 4, affine)
    g = _rand(8)
    ds = torch.randn(2, 41, 520, device=DEV, generator=g).bfloat16()
    dh = torch.randn(2, 41, 520, device=DEV, generator=g).bfloat16() if norm is not None else None
    _check_norm(a, f"{norm}/{post}/{mod}/{affine}", ds, dh, norm=norm, post_norm=post, residual_scale=0.5,
                branch_scale=1.7, eps=1e-5)


@pytest.mark.parametrize("only", ["ds", "dh"])
def test_gated_norm_one_gradient(only):
    a = _norm_inputs(12, 1, 65, 1536, "fp32", None, "rms", "layer")
    d = torch.randn(1, 65, 1536, device=DEV, generator=_rand(9))
    _check_norm(a, only, **{only: d}, norm="rms", post_norm="layer")


def test_gated_norm_without_branch():
    """norm + modulation alone: h, no stream."""
    a = _norm_inputs(13, 2, 37, 768, "bf16", "fp32")
    a = {k: v for k, v in a.items() if k not in ("y", "gate", "post_weight")}
    dh = torch.randn(2, 37, 768, device=DEV, generator=_rand(10)).bfloat16()
    _check_norm(a, "no branch", None, dh)


def test_gated_norm_strides_and_ragged_rows():
    """x a slice of a wider tensor, y transposed, modulations slices of one projection or expanded over the batch, tokens that
    do not divide into the rows (the last row short, one row past the end with zero gradients)."""
    g = _rand(14)
    b, n, c = 2, 22, 512
    x = torch.randn(b, n + 5, c + 64, device=DEV, generator=g).bfloat16()[:, 3:n + 3, 64:]
    y = torch.randn(n, b, c, device=DEV, generator=g).bfloat16().transpose(0, 1)
    six = torch.randn(b, 5, 6, c, device=DEV, generator=g)
    a = {"x": x, "y": y, "gate": six[:, :, 2], "shift": six[:, :, 3],
         "scale": torch.randn(1, 1, c, device=DEV, generator=g).expand(b, 5, c)}
    ds, dh = (torch.randn(b, n, c, device=DEV, generator=g).bfloat16() for _ in range(2))
    _check_norm(a, "strides", ds, dh, group_len=6)   # rows of 6, 6, 6, 4 and 0 tokens
    from lingbot_world_v2_realtime_amd import gated_norm
    leaf = {k: v.detach().requires_grad_() for k, v in a.items()}
    s, h = gated_norm(**leaf, group_len=6)
    d = torch.autograd.grad([s, h], [leaf["gate"], leaf["shift"], leaf["scale"]], [ds, dh])
    assert all(not t[:, 4].any() for t in d)
    # gradients of an expanded leaf's own memory, and of outputs summed (expanded gradients)
    one = torch.randn(c, device=DEV, generator=g, requires_grad=True)
    gated_norm(x, y, gate=one.expand(b, 5, c), group_len=6)[0].sum().backward()
    assert one.grad.shape == (c,) and bool(one.grad.isfinite().all())


def test_gated_norm_a_row_for_each_token():
    """Modulation rows of one token each, more of them (with the batch) than a grid's second dimension has."""
    a = _norm_inputs(24, 3, 37, 520, "bf16", "fp32", rows=37)
    g = _rand(25)
    ds, dh = (torch.randn(3, 37, 520, device=DEV, generator=g).bfloat16() for _ in range(2))
    _check_norm(a, "a row a token", ds, dh)
    a = _norm_inputs(26, 300, 250, 16, "fp32", rows=250)
    ds, dh = (torch.randn(300, 250, 16, device=DEV, generator=g) for _ in range(2))
    _check_norm({k: v for k, v in a.items() if k in ("x", "y", "gate", "shift", "scale")}, "75000 rows", ds, dh)


def test_gated_norm_unaligned_rows():
    """Rows that start at any element: the value-by-value form."""
    g = _rand(15)
    x = torch.randn(3, 9, 257, device=DEV, generator=g).half()[:, :, 1:]
    y = torch.randn(3, 9, 259, device=DEV, generator=g).half()[:, :, 3:]
    w = torch.randn(257, device=DEV, generator=g).half()[1:]
    ds, dh = (torch.randn(3, 9, 256, device=DEV, generator=g).half() for _ in range(2))
    _check_norm({"x": x, "y": y, "weight": w, "gate": w}, "unaligned", ds, dh, norm="rms", post_norm="rms")


def test_gated_norm_mixed_vectors_and_empty():
    from lingbot_world_v2_realtime_amd import gated_norm
    a = _norm_inputs(16, 1, 20, 256, "bf16", "bf16")
    a["gate"], a["scale"] = a["gate"].float(), a["scale"].float()
    leaf = {k: v.detach().requires_grad_() for k, v in a.items()}
    s, h = gated_norm(**leaf)
    d = torch.autograd.grad([s, h], list(leaf.values()), [torch.ones_like(s), torch.ones_like(h)])
    assert all(g.dtype == v.dtype and g.shape == v.shape for g, v in zip(d, leaf.values()))
    empty = {k: (v[:, :0] if k in ("x", "y") else v).detach().requires_grad_() for k, v in a.items()}
    s, h = gated_norm(**empty)
    assert s.shape == h.shape == (1, 0, 256)
    d = torch.autograd.grad([s, h], list(empty.values()), [torch.ones_like(s), torch.ones_like(h)])
    assert all(not g.any() for g in d)


def test_gated_norm_constant_and_nonfinite_rows():
    """A row of equal values (variance zero) gives bias and shift; a NaN or an infinity stays in its row."""
    from lingbot_world_v2_realtime_amd import gated_norm
    a = _norm_inputs(17, 1, 12, 640, "bf16", "fp32", rows=2)
    a["x"][0, 3], a["y"][0, 3] = 2.5, 0.0
    clean = gated_norm(**a)
    want = a["bias"] * (1 + a["scale"][0, 0]) + a["shift"][0, 0]
    assert torch.equal(clean[1][0, 3], want.bfloat16())
    bad = {k: v.clone() for k, v in a.items()}
    bad["x"][0, 5, 100], bad["y"][0, 7, 3] = float("nan"), float("inf")
    out = gated_norm(**bad)
    rows = [i for i in range(12) if i not in (5, 7)]
    for o, c in zip(out, clean):
        assert torch.equal(o[0, rows], c[0, rows])
    assert bool(out[1][0, 5].isnan().all())


def test_gated_norm_same_bits_and_partial_gradients():
    """Two runs give the same bits, and a gradient does not change with which others are asked for."""
    from lingbot_world_v2_realtime_amd import kernels
    a = _norm_inputs(18, 2, 500, 1536, "bf16", "fp32", "layer", "rms", rows=3)
    g = _rand(19)
    ds, dh = (torch.randn(2, 500, 1536, device=DEV, generator=g).bfloat16() for _ in range(2))
    kw = dict(norm="layer", post_norm="rms")
    whole = kernels.gated_norm_bwd(a["x"], ds, dh, **{k: v for k, v in a.items() if k != "x"}, **kw)
    assert set(whole) == set(a)
    for name in a:
        one = kernels.gated_norm_bwd(a["x"], ds, dh, **{k: v for k, v in a.items() if k != "x"}, **kw, wants=(name,))
        assert list(one) == [name] and torch.equal(one[name], whole[name]), name


def _replays(make, change, n=3):
    """make() captured into a graph, replayed n times with other inputs (change(i)) and eager work between."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        make()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = make()
    for i in range(n):
        change(i)
        want = [w.clone() for w in make()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, want):
            assert torch.equal(o, w), f"replay {i}"


def test_gated_norm_in_a_graph():
    from lingbot_world_v2_realtime_amd import kernels
    a = _norm_inputs(20, 1, 130, 1536, "bf16", "fp32")
    g = _rand(21)
    ds, dh = (torch.randn(1, 130, 1536, device=DEV, generator=g).bfloat16() for _ in range(2))
    rest = {k: v for k, v in a.items() if k != "x"}

    def make():
        return [*kernels.gated_norm(**a), *kernels.gated_norm_bwd(a["x"], ds, dh, **rest).values()]

    _replays(make, lambda i: a["x"].add_(0.25))


def test_training_step_in_a_graph():
    """Forward and backward through autograd, captured and replayed."""
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    a = {k: v.requires_grad_() for k, v in _norm_inputs(27, 1, 70, 512, "bf16", "fp32").items()}
    rope, pos = Rotary.build(128, DEV, pairs="half"), torch.arange(70, device=DEV)

    def make():
        s, h = gated_norm(**a)
        q, _ = rotary_embed(h.view(1, 70, 4, 128), None, pos, rope)
        return torch.autograd.grad((s, q), list(a.values()), (torch.ones_like(s), torch.ones_like(q)))

    _replays(make, lambda i: a["x"].detach().add_(0.25))


def test_calls_on_another_stream():
    """Each operator on a side stream, ordered only by that stream."""
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, kernels, rotary_embed
    a = _norm_inputs(22, 1, 400, 1536, "bf16", "fp32")
    q = torch.randn(1, 400, 4, 128, device=DEV).bfloat16()
    rope = Rotary.build(128, DEV)
    w4 = kernels.quant_w4(torch.randn(256, 1536, device=DEV))
    want = [*gated_norm(**a), rotary_embed(q, None, 5, rope)[0], kernels.gemm_w4(a["x"][0], *w4)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [*gated_norm(**a), rotary_embed(q, None, 5, rope)[0], kernels.gemm_w4(a["x"][0], *w4)]
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_gated_norm_refusals():
    from lingbot_world_v2_realtime_amd import gated_norm
    a = _norm_inputs(23, 2, 12, 64, rows=3)
    x, y = a["x"], a["y"]
    for bad in (dict(y=y[:, :5]), dict(gate=a["gate"][:1]), dict(gate=a["gate"][:, :2], group_len=5),
                dict(weight=a["weight"][:32]), dict(scale=a["scale"][:, :, ::2]), dict(shift=a["shift"][:, :2]),
                dict(norm="batch"), dict(post_norm="none"), dict(group_len=3, gate=None, shift=None, scale=None),
                dict(y=None), dict(norm=None), dict(x=x.transpose(1, 2)), dict(x=x[0])):
        with pytest.raises(ValueError):
            gated_norm(**{**a, **bad})
    with pytest.raises(TypeError):
        gated_norm(x, y.float())
    with pytest.raises(TypeError):
        gated_norm(x, y, gate=torch.ones(64, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        gated_norm(x, norm=None)
    with pytest.raises(ValueError, match="different devices"):
        gated_norm(x, y, gate=torch.ones(64, dtype=torch.bfloat16))


def test_gradients_once_and_transforms():
    """A second derivative, forward-mode tangents and torch.func transforms are refused, not answered wrongly; a tensor changed
    after the call is noticed by the gradient."""
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    x = torch.randn(1, 4, 64, device=DEV, requires_grad=True)
    rope = Rotary.build(64, DEV)
    calls = (lambda t: gated_norm(t), lambda t: rotary_embed(t.view(1, 4, 1, 64), None, 0, rope)[0].view(1, 4, 64))
    for f in calls:
        (g,) = torch.autograd.grad(f(x).sum(), x)
        assert bool(g.isfinite().all())
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(f(x).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x.detach(),), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x.detach())
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda t: f(t))(torch.randn(3, 1, 4, 64, device=DEV))
    y = x * 1.0
    out = gated_norm(y)
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    q = torch.randn(1, 4, 2, 64, device=DEV, requires_grad=True)
    z = q * 1.0
    w = z.square().sum()
    with torch.no_grad():
        rotary_embed(z, None, 0, rope, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.backward()
    with torch.inference_mode():
        t = torch.randn(1, 4, 2, 64, device=DEV)
        assert rotary_embed(t, None, 0, rope, inplace=True)[0] is not None and gated_norm(t.view(1, 8, 64)).shape == (1, 8, 64)


# ---------------------------------------------------------------- rotary


def _check_rotary(q, k, pos, rope, what, layout="NHD", train=True):
    from lingbot_world_v2_realtime_amd import rotary_embed
    leaves = [t.detach().requires_grad_(train) for t in (q, k) if t is not None]
    out = rotary_embed(leaves[0], leaves[1] if k is not None else None, pos, rope, layout)
    assert (out[1] is None) == (k is None)
    nhd = (lambda t: t) if layout == "NHD" else (lambda t: t.transpose(1, 2))
    n = nhd(q).shape[1]
    p = pos if isinstance(pos, torch.Tensor) else torch.arange(n, device=DEV) + pos
    args = dict(freq=rope.freq, axis=rope.axis, pairs=rope.pairs, factor=rope.factor)
    k_of = 12 + float(p.abs().max()) * float(rope.freq.max()) * 2.0 ** -27   # (the 64-bit angle's own rounding)
    g = _rand(31)
    for x, o in zip(leaves, out):
        assert o.shape == x.shape and o.dtype == x.dtype
        _within(nhd(o.detach()), block.rotary(nhd(x), p, **args), what, k_of)
        rest = nhd(o)[..., 2 * rope.freq.shape[0]:]
        assert torch.equal(rest, nhd(x)[..., 2 * rope.freq.shape[0]:])
    if not train:
        return
    d = [torch.randn(x.shape, device=DEV, generator=g).to(x.dtype) for x in leaves]
    for x, gr, dd in zip(leaves, torch.autograd.grad([o for o in out if o is not None], leaves, d), d):
        _within(nhd(gr), block.rotary(nhd(dd), p, **args, inverse=True), f"{what}: gradient", k_of)


def _qk(seed, b, n, hq, hk, d, dtype="bf16"):
    g = _rand(seed)
    q = torch.randn(b, n, hq, d, device=DEV, generator=g).to(DT[dtype])
    return q, torch.randn(b, n, hk, d, device=DEV, generator=g).to(DT[dtype]) if hk else None


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("b,n,hq,hk,d,rot", [(1, 1, 1, 0, 2, 2), (1, 7, 3, 1, 128, 128), (2, 65, 8, 2, 128, 64),
                                             (3, 5, 4, 4, 96, 24), (1, 33, 2, 2, 80, 70), (2, 3, 1, 1, 7, 6),
                                             (1, 3, 5, 1, 512, 512), (40, 1, 12, 2, 128, 128)])
def test_rotary_sizes(dtype, pairs, b, n, hq, hk, d, rot):
    from lingbot_world_v2_realtime_amd import Rotary
    q, k = _qk(n + d, b, n, hq, hk, d, dtype)
    pos = torch.randint(0, 5000, (b, n), device=DEV, generator=_rand(1))
    _check_rotary(q, k, pos, Rotary.build(rot, DEV, pairs=pairs), f"{dtype} {pairs} {b}x{n}x{hq}/{hk}x{d}/{rot}")


def test_rotary_positions():
    """Each form of positions, far ones (past 32 bits), negative ones, the same one twice, strided."""
    from lingbot_world_v2_realtime_amd import Rotary, grid_positions
    q, k = _qk(41, 2, 24, 4, 2, 128)
    one, three = Rotary.build(128, DEV), Rotary.build(128, DEV, sections=(22, 21, 21))
    ramp = Rotary.build(128, DEV, pairs="half", scaling="ramp", stretch=8.0, trained_len=4096)
    i64 = torch.randint(-1000000, 1000000, (2, 24), device=DEV, generator=_rand(2))
    far = torch.full((24,), (1 << 33) + 7, device=DEV)
    for pos, rope in ((0, one), (123456789, one), (-5, ramp), (i64, one), (i64.int(), ramp), (i64[0], one), (far, one),
                      (torch.zeros(24, dtype=torch.int32, device=DEV), one), (i64.t().contiguous().t(), ramp),
                      (grid_positions((2, 3, 4), 1000, DEV), three),
                      (torch.randint(0, 9999, (2, 24, 5), device=DEV, generator=_rand(3))[:, :, 1:4], three)):
        _check_rotary(q, k, pos, rope, f"positions {getattr(pos, 'dtype', pos)}")


def test_rotary_layouts_strides_and_inplace():
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    rope = Rotary.build(64, DEV, pairs="half")
    q, k = _qk(42, 2, 30, 6, 2, 128)
    _check_rotary(q.transpose(1, 2), k.transpose(1, 2), 9, rope, "HND views", "HND")
    _check_rotary(q.transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous(), 9, rope, "HND", "HND")
    fused = torch.randn(2, 30, 10 * 128, device=DEV, generator=_rand(4)).bfloat16()   # q, k, v of one projection
    qv, kv = fused[..., :768].unflatten(-1, (6, 128)), fused[..., 768:1024].unflatten(-1, (2, 128))
    _check_rotary(qv, kv, 9, rope, "views of a projection")
    shared = torch.randn(2, 30, 1, 128, device=DEV, generator=_rand(5)).bfloat16().expand(2, 30, 6, 128)
    _check_rotary(shared, k, 9, rope, "one head shared by six")
    odd = torch.randn(2, 30, 3, 131, device=DEV, generator=_rand(6)).bfloat16()[..., 3:]
    _check_rotary(odd, None, 9, rope, "unaligned")
    want = rotary_embed(qv, kv, 9, rope)
    rest = fused[..., 1024:].clone()
    got = rotary_embed(qv, kv, 9, rope, inplace=True)
    assert got[0].data_ptr() == qv.data_ptr() and all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(fused[..., 1024:], rest)
    with pytest.raises(ValueError):
        rotary_embed(shared, None, 9, rope, inplace=True)
    from lingbot_world_v2_realtime_amd import kernels
    with pytest.raises(ValueError, match="share their memory"):
        rotary_embed(q, q, 9, rope, inplace=True)
    with pytest.raises(ValueError, match="share their memory"):
        kernels.rotary(q, q.clone(), 9, rope.freq, q_out=q, k_out=q)
    with pytest.raises(ValueError, match="share their memory"):
        kernels.rotary(q, k, 9, rope.freq, k_out=q[:, :, :2])
    with pytest.raises(ValueError):
        rotary_embed(q.detach().requires_grad_(), k, 9, rope, inplace=True)


def test_rotary_one_gradient_and_empty():
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    rope = Rotary.build(128, DEV)
    q, k = _qk(43, 1, 17, 4, 2, 128, "fp32")
    dk = torch.randn_like(k)
    for leaf in ("q", "k", "only k's output"):
        lq, lk = q.detach().requires_grad_(leaf != "k"), k.detach().requires_grad_(leaf != "q")
        oq, ok = rotary_embed(lq, lk, 3, rope)
        (ok.mul(dk).sum() + (0 if leaf == "only k's output" else oq.sum())).backward()
        if leaf != "q":
            _within(lk.grad, block.rotary(dk, torch.arange(3, 20, device=DEV), rope.freq, inverse=True), leaf, 13)
        assert (lq.grad is None) == (leaf != "q")
    for n, h in ((0, 4), (5, 0)):
        if h == 0:
            continue
        oq, ok = rotary_embed(q[:, :n], k[:, :n], 0, rope)
        assert oq.shape == (1, n, 4, 128) and ok.shape == (1, n, 2, 128)


def test_rotary_matches_the_fused_prologue():
    """The model's three axes: the same rotation as the quantising prologue's table (which rounds after a norm of weight
    one, here on rows of unit mean square)."""
    from lingbot_world_v2_realtime_amd import Rotary, grid_positions, rotary_embed
    from lingbot_world_v2_realtime_amd.layers.prologue import ChunkRope, norm_rope, rope_freqs
    x = torch.where(torch.rand(1, 60, 2 * 128, device=DEV, generator=_rand(7)) < 0.5, 1.0, -1.0).bfloat16()
    got = rotary_embed(x.unflatten(-1, (2, 128)), None, grid_positions((3, 4, 5), 17, DEV),
                       Rotary.build(128, DEV, sections=(22, 21, 21)))[0]
    want = norm_rope(x, 2, torch.ones(256, device=DEV).bfloat16(), 0.0, ChunkRope(rope_freqs(DEV), 4, 5, 17))
    # equal up to a value at a rounding's border: one step of a value of 2 at most
    assert (got.float() - want.float()).abs().max().item() <= 2.0 ** -7


def test_rotary_in_a_graph():
    from lingbot_world_v2_realtime_amd import Rotary, kernels
    rope = Rotary.build(128, DEV, sections=(22, 21, 21))
    q, k = _qk(44, 2, 50, 4, 2, 128)
    pos = torch.randint(0, 100, (2, 50, 3), device=DEV)
    _replays(lambda: list(kernels.rotary(q, k, pos, rope.freq, rope.axis)), lambda i: pos.add_(1))


def test_rotary_refusals():
    from lingbot_world_v2_realtime_amd import Rotary, kernels, rotary_embed
    rope, three = Rotary.build(128, DEV), Rotary.build(128, DEV, sections=(22, 21, 21))
    q, k = _qk(45, 2, 6, 4, 2, 128)
    pos = torch.zeros(2, 6, dtype=torch.int64, device=DEV)
    for bad in (lambda: rotary_embed(q, k[:, :5], 0, rope), lambda: rotary_embed(q, k[..., :64], 0, rope),
                lambda: rotary_embed(q[..., :64], None, 0, rope), lambda: rotary_embed(q, k, pos[:, :5], rope),
                lambda: rotary_embed(q, k, pos, three), lambda: rotary_embed(q, k, 3, three),
                lambda: rotary_embed(q, k, pos[..., None], rope), lambda: rotary_embed(q[0], None, 0, rope),
                lambda: rotary_embed(q, k, pos.cpu(), rope), lambda: rotary_embed(q, k, 0, rope, "LHD"),
                lambda: kernels.rotary(q, k, 0, rope.freq.float()), lambda: kernels.rotary(q, k, 0, rope.freq, pairs="x"),
                lambda: kernels.rotary(q, None, 0, rope.freq, k_out=k),
                lambda: kernels.rotary(q, None, 0, rope.freq, q_out=q.transpose(0, 1)),
                lambda: rotary_embed(q.transpose(2, 3), None, 0, rope)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: rotary_embed(q, k.half(), 0, rope), lambda: rotary_embed(q, k, pos.float(), rope),
                lambda: rotary_embed(q.double(), None, 0, rope), lambda: rotary_embed(q, k, 0.5, rope)):
        with pytest.raises(TypeError):
            bad()


# ---------------------------------------------------------------- 4-bit linears


@pytest.mark.parametrize("fmt,zeros", [("int4", False), ("int4", True), ("fp4", False)])
@pytest.mark.parametrize("n,k,group", [(16, 128, 128), (1, 1, 32), (37, 300, 64), (160, 1536, 32), (33, 129, 128)])
def test_quant_w4(fmt, zeros, n, k, group):
    """The kernel's codes, scales and zeros, bit for bit, from bf16 and fp32 weights, a zero group and tiny values."""
    from lingbot_world_v2_realtime_amd import kernels
    w = torch.randn(n, k, device=DEV, generator=_rand(n + k))
    w[0, :group] = 0
    w[-1, :group] *= 1e-39 if n > 1 else 1.0
    full = torch.zeros(-(-n // 16) * 16, -(-k // 128) * 128, device=DEV)
    for src in (w, w.bfloat16()):
        full[:n, :k] = src.float()
        # (on the CPU: torch divides by a number through its reciprocal on the GPU)
        codes, scale, zero = (t if t is None else t.to(DEV) for t in block.quant_w4(full.cpu(), group, fmt, zeros))
        w4, sc, z = kernels.quant_w4(src, group, fmt, zeros)
        assert torch.equal(block.unpack_scale(sc), scale)
        assert (z is None) if zero is None else torch.equal(block.unpack_scale(z), zero)
        got = block.unpack_w4(w4, fmt)
        # (a code of a group without a scale stands for zero whatever it is)
        live = scale.float().repeat_interleave(group, 1) > 0
        # minus zero and zero are one value of fp4
        same = (got == codes) | ((fmt == "fp4") & ((got | codes) & 7 == 0))
        assert bool((same | ~live).all())


def _w4(seed, n, k, group, fmt, zeros):
    """Weights at every code, random scales and zeros, and their values in 64 bits."""
    from lingbot_world_v2_realtime_amd import kernels
    g = _rand(seed)
    codes = torch.randint(0, 16, (n, k), device=DEV, generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scale = (torch.rand(n, groups, device=DEV, generator=g) + 0.1).bfloat16()
    zero = torch.randint(0, 16, (n, groups), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
    pad = torch.zeros(n, groups * group, dtype=torch.uint8, device=DEV)
    pad[:, :k] = codes
    value = block.w4_values(pad, scale, zero, fmt)[:, :k]
    # what the products add: fp4 the values, integer codes up to 16 + 15 and their offset of up to 16 + 15 steps
    steps = scale.double().repeat_interleave(group, 1)[:, :k] * (62 if fmt == "int4" else 6)
    return kernels.pack_w4(codes, scale, zero, fmt), value, steps


def _check_w4(m, n, k, group, fmt, zeros, dtype, bias, x=None):
    from lingbot_world_v2_realtime_amd import kernels
    packed, value, steps = _w4(n + k, n, k, group, fmt, zeros)
    g = _rand(m)
    x = torch.randn(m, k, device=DEV, generator=g).to(DT[dtype]) if x is None else x
    b = torch.randn(n, device=DEV, generator=g).to(DT[dtype]) if bias else None
    out = kernels.gemm_w4(x, *packed, b, out_features=n, fmt=fmt)
    want, _ = block.w4_linear(x, value, b)
    mag = x.double().abs() @ steps.t().contiguous()
    _within(out, (want, mag + want.abs()), f"{m}x{n}x{k} group {group} {fmt} {zeros} {dtype}", k / 16 + 24)


# every kernel and tile, with rows, columns and K that end inside a tile: 16 x 16, 16 x 32, 16 x 48 and 32 x 48 (by the
# workgroups they give, and by the rows), 64 x 256 (from 128 of those on)
W4_SIZES = [(1, 16, 128), (1, 1, 1), (3, 37, 300), (16, 64, 1536), (17, 48, 256), (33, 100, 520), (65, 130, 384),
            (130, 257, 640), (300, 144, 1000), (2, 1536, 8960), (129, 16, 128), (100, 1203, 264), (70, 4004, 392),
            (300, 1601, 136), (450, 5204, 520), (1030, 2310, 256), (100, 700, 264), (65, 1000, 1536),
            (9, 12400, 136), (20, 32800, 128)]


@pytest.mark.parametrize("m,n,k", W4_SIZES)
@pytest.mark.parametrize("fmt,zeros,group,dtype", [("int4", False, 128, "bf16"), ("int4", True, 64, "fp16"),
                                                   ("int4", True, 32, "bf16"), ("fp4", False, 32, "fp16"),
                                                   ("fp4", False, 128, "bf16")])
def test_gemm_w4(m, n, k, fmt, zeros, group, dtype):
    _check_w4(m, n, k, group, fmt, zeros, dtype, bias=m % 2 == 1)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_gemm_w4_groups(m, group):
    for fmt, zeros in (("int4", False), ("int4", True), ("fp4", False)):
        _check_w4(m, 80, 448, group, fmt, zeros, "bf16", True)


def test_gemm_w4_strides():
    """Rows of a wider tensor, one row for all (stride 0), unaligned rows, an empty x."""
    from lingbot_world_v2_realtime_amd import kernels
    g = _rand(51)
    wide = torch.randn(70, 400, device=DEV, generator=g).bfloat16()
    _check_w4(70, 48, 256, 64, "int4", True, "bf16", True, x=wide[:, 8:264])
    _check_w4(70, 48, 256, 64, "int4", True, "bf16", True, x=wide[:, 3:259])
    _check_w4(20, 48, 256, 64, "fp4", False, "bf16", True, x=wide[:1, :256].expand(20, 256))
    _check_w4(9, 48, 250, 64, "fp4", False, "bf16", True, x=wide[:9, :250])
    packed, _, _ = _w4(3, 48, 256, 64, "int4", True)
    assert kernels.gemm_w4(wide[:0, :256], *packed).shape == (0, 48)
    # weights inside a larger buffer, at any address
    moved = [torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape) for t in packed]
    assert torch.equal(kernels.gemm_w4(wide[:, :256], *moved), kernels.gemm_w4(wide[:, :256], *packed))


def test_gemm_w4_rows_do_not_mix():
    """A row's result is the same bits alone as among others of its kernel, and a NaN stays in its row."""
    from lingbot_world_v2_realtime_amd import kernels
    packed, _, _ = _w4(52, 64, 512, 128, "int4", True)
    for m in (16, 64, 300, 10240):
        x = torch.randn(m, 512, device=DEV, generator=_rand(53)).bfloat16()
        clean = kernels.gemm_w4(x[:m], *packed)
        bad = x[:m].clone()
        bad[m // 2, 77] = float("nan")
        out = kernels.gemm_w4(bad, *packed)
        rows = [i for i in range(m) if i != m // 2]
        assert torch.equal(out[rows], clean[rows]) and bool(out[m // 2].isnan().all())
        assert torch.equal(kernels.gemm_w4(x[:m], *packed), clean)


def test_gemm_w4_in_a_graph():
    from lingbot_world_v2_realtime_amd import kernels
    packed, _, _ = _w4(54, 144, 1536, 128, "int4", False)
    x = torch.randn(300, 1536, device=DEV).bfloat16()
    _replays(lambda: [kernels.gemm_w4(x[:m], *packed) for m in (1, 40, 300)], lambda i: x.add_(0.5))


@pytest.mark.parametrize("fmt,zeros", [("int4", False), ("int4", True), ("fp4", False)])
def test_w4_linear(fmt, zeros):
    """The module: weights quantised from an nn.Linear, leading dims, activation types, biases with a gradient."""
    from lingbot_world_v2_realtime_amd.layers.linear import W4Linear, convert_to_w4
    torch.manual_seed(0)
    lin = torch.nn.Linear(1536, 1040).to(DEV).bfloat16()
    mod = W4Linear(lin, 64, fmt, zeros)
    sc, z = block.unpack_scale(mod.w4_scale), None if mod.w4_zero is None else block.unpack_scale(mod.w4_zero)
    value = block.w4_values(block.unpack_w4(mod.w4, fmt), sc, z, fmt)[:1040, :1536]
    step = sc.double().repeat_interleave(64, 1)[:1040, :1536]
    assert bool(((value - lin.weight.double()).abs() <= step * (1.05 if fmt == "fp4" else 0.55)).all())
    x = torch.randn(2, 3, 1536, device=DEV).bfloat16()
    steps = step * (62 if fmt == "int4" else 6)
    with torch.no_grad():
        y = mod(x)
        assert y.shape == (2, 3, 1040) and y.dtype == torch.bfloat16
        want, _ = block.w4_linear(x.reshape(6, 1536), value, lin.bias)
        mag = x.reshape(6, 1536).double().abs() @ steps.t().contiguous()
        _within(y.reshape(6, 1040), (want, mag + want.abs()), "module", 1536 / 16 + 24)
        assert torch.equal(mod(x.float()), y) and mod(x.half()).dtype == torch.float16
        assert torch.equal(mod(x[0, 0]), mod(x[:1, 0])[0])
    y = mod(x)
    y.float().sum().backward()
    assert torch.equal(lin.bias.grad, torch.full_like(lin.bias, 6.0))
    with pytest.raises(RuntimeError, match="no gradient"):
        mod(x.requires_grad_())
    net = torch.nn.Sequential(torch.nn.Linear(1536, 1024), torch.nn.Linear(1024, 8)).to(DEV)
    assert convert_to_w4(net, fmt=fmt, zeros=zeros) == (1, 2)
    # casts of the module leave the weights alone; a copy through its state is the same module
    scale, x = net[0].w4_scale.clone(), torch.randn(5, 1536, device=DEV).half()
    with torch.no_grad():
        want = net.half()[0](x)
        assert torch.equal(net[0].w4_scale, scale) and want.dtype == torch.float16
        other = W4Linear(torch.nn.Linear(1536, 1024).to(DEV), 128, fmt, zeros).half()
        other.load_state_dict(net[0].state_dict())
        assert torch.equal(other(x), want)


def test_w4_refusals():
    from lingbot_world_v2_realtime_amd import kernels
    x = torch.zeros(3, 256, device=DEV, dtype=torch.bfloat16)
    (w4, scale, zero), _, _ = _w4(55, 40, 256, 64, "int4", True)
    for bad in (dict(w4=w4[:2]), dict(w4=w4.int()), dict(scale=scale.float()), dict(scale=scale[..., :1].contiguous()),
                dict(zero=zero[:, :1]), dict(zero=zero.int()), dict(x=x[:, :100].contiguous()), dict(x=x.t()),
                dict(bias=torch.zeros(48, device=DEV)), dict(bias=x[0, :40]), dict(out_features=60), dict(fmt="fp4"),
                dict(fmt="int3"), dict(x=x[0]), dict(w4=w4.cpu())):
        with pytest.raises(ValueError):
            kernels.gemm_w4(**{"x": x, "w4": w4, "scale": scale, "zero": zero, **bad})
    for bad in (dict(group=16), dict(fmt="nf4"), dict(fmt="fp4", zeros=True), dict(w=x[0]), dict(w=x[:0])):
        with pytest.raises(ValueError):
            kernels.quant_w4(**{"w": x, **bad})
    with pytest.raises(TypeError):
        kernels.quant_w4(x.half())


# ---------------------------------------------------------------- together


def test_block_step():
    """A block's path through the operators: the time embedding's row through a 4-bit linear to the modulation, the gated norm,
    4-bit q / k projections, rotary positions, attention, and the gated residual, against the same in 64 bits on the same
    quantised weights. Each stage is checked on the inputs the stage before gave it."""
    from lingbot_world_v2_realtime_amd import Rotary, flash_attention, gated_norm, grid_positions, rotary_embed
    from lingbot_world_v2_realtime_amd.layers.linear import W4Linear
    torch.manual_seed(3)
    c, heads, f, n = 256, 2, 2, 2 * 30
    mod = W4Linear(torch.nn.Linear(c, 6 * c).to(DEV).bfloat16())
    qkv = W4Linear(torch.nn.Linear(c, 3 * c).to(DEV).bfloat16(), 32, "fp4")
    with torch.no_grad():
        e = mod(torch.randn(1, f, c, device=DEV).bfloat16()).view(1, f, 6, c)
        x = torch.randn(1, n, c, device=DEV).bfloat16()
        h = gated_norm(x, shift=e[:, :, 0], scale=e[:, :, 1])
        _within(h, block.gated_norm(x, shift=e[:, :, 0], scale=e[:, :, 1])[1], "first norm", 96)
        q, k, v = qkv(h).view(1, n, 3, heads, 128).unbind(2)
        rope, pos = Rotary.build(128, DEV, sections=(22, 21, 21)), grid_positions((f, 5, 6), 3, DEV)
        q2, k2 = rotary_embed(q, k, pos, rope)
        for a, b in ((q, q2), (k, k2)):
            _within(b, block.rotary(a, pos, rope.freq, rope.axis), "rotary", 13)
        y = flash_attention(q2, k2, v).reshape(1, n, c)
        kw = dict(gate=e[:, :, 2], shift=e[:, :, 3], scale=e[:, :, 4])
        s, h2 = gated_norm(x, y, **kw)
        ws, wh, _ = block.gated_norm(x, y, **kw)
        _within(s, ws, "stream", 96)
        _within(h2, wh, "second norm", 96)


# ---------------------------------------------------------------- the largest launches


def _tail(t, rows):
    return t[:, -rows:]


def test_gated_norm_more_threads_than_a_grid_dimension():
    """2^26 + 5 narrow rows, a wave each: more than the 2^32 threads that one grid dimension holds. A modulation row for every
    token, so its gradient's workgroups are as many."""
    from lingbot_world_v2_realtime_amd import kernels
    n, c, last = 2 ** 26 + 5, 8, 4099
    g = _rand(60)
    x, shift, dh = (torch.randn(1, n, c, device=DEV, generator=g, dtype=torch.bfloat16) for _ in range(3))
    print("rows", n, "forward", flush=True)
    h = kernels.gated_norm(x, shift=shift, norm="rms")[1]
    for part in (slice(0, last), slice(n - last, n), slice(2 ** 22 - 70, 2 ** 22 + 70)):
        _within(h[:, part], block.gated_norm(x[:, part], shift=shift[:, part], norm="rms")[1], f"h {part}", 96)
    del h
    print("rows", n, "backward", flush=True)
    d = kernels.gated_norm_bwd(x, None, dh, shift=shift, norm="rms", wants=("x", "shift"))
    assert torch.equal(d["shift"], dh)   # each the sum of one row
    one = kernels.gated_norm_bwd(_tail(x, last), None, _tail(dh, last).contiguous(), shift=_tail(shift, last), norm="rms",
                                 wants=("x",))
    assert torch.equal(_tail(d["x"], last), one["x"])


def test_rotary_more_threads_than_a_grid_dimension():
    from lingbot_world_v2_realtime_amd import kernels
    n, last = 2 ** 27 + 11, 4099
    q = torch.randn(1, n, 1, 2, device=DEV, generator=_rand(61), dtype=torch.bfloat16)
    freq = torch.tensor([0.7], dtype=torch.float64, device=DEV)
    print("tokens", n, flush=True)
    out = kernels.rotary(q, None, 5, freq)[0]
    for part in (slice(0, last), slice(n - last, n)):
        pos = torch.arange(5 + part.start, 5 + part.stop, device=DEV)
        _within(out[:, part], block.rotary(q[:, part], pos, freq), f"{part}", 13)


def test_flags_numbers_and_overlaps():
    """Flags of any truth value; factors and frequencies that would lose their gradient, and outputs that overlap their input,
    are refused."""
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, kernels, rotary_embed
    rope = Rotary.build(64, DEV)
    q, _ = _qk(62, 1, 9, 2, 1, 64)
    want = rotary_embed(q, None, 0, rope)[0]
    buf = torch.zeros(1, 10, 2, 64, device=DEV, dtype=q.dtype)
    buf[:, :9] = q
    with pytest.raises(ValueError, match="overlaps"):
        kernels.rotary(buf[:, :9], None, 0, rope.freq, q_out=buf[:, 1:])
    assert rotary_embed(q, None, 0, rope, inplace=1)[0].data_ptr() == q.data_ptr() and torch.equal(q, want)
    learned = Rotary(rope.freq.clone().requires_grad_())
    with pytest.raises(ValueError, match="freq"):
        rotary_embed(q, None, 0, learned)
    with torch.no_grad():
        assert torch.equal(rotary_embed(q, None, 0, learned)[0], rotary_embed(q, None, 0, rope)[0])
    x = torch.randn(1, 4, 64, device=DEV)
    for name in ("residual_scale", "branch_scale", "eps"):
        with pytest.raises(TypeError, match="gradient"):
            gated_norm(x, x, **{name: torch.ones((), requires_grad=True)})
    assert kernels.gated_norm(x, x, want_stream=1)[0] is not None and kernels.gated_norm(x, x, want_stream=0)[0] is None
    grad = torch._neg_view(torch.randn(1, 4, 64, device=DEV))
    leaf = x.clone().requires_grad_()
    got = torch.autograd.grad(gated_norm(leaf), leaf, grad)[0]
    assert torch.equal(got, torch.autograd.grad(gated_norm(leaf), leaf, grad.resolve_neg())[0])


def test_w4_linear_takes_floating_point_rows():
    from lingbot_world_v2_realtime_amd.layers.linear import W4Linear
    mod = W4Linear(torch.nn.Linear(128, 16).to(DEV))
    with torch.no_grad():
        with pytest.raises(TypeError, match="floating-point"):
            mod(torch.ones(2, 128, device=DEV, dtype=torch.int64))
        assert mod(torch.ones(0, 128, device=DEV)).shape == (0, 16)
