"""Calls that the block operators' documentation allows at the edges of their sizes, layouts and types, on the GPU against
the definitions in 64 bits (oracle/block.py), with the bounds of test_gpu_block.py."""
import pytest
import torch

from oracle import block
from test_gpu_block import DEV, DT, _check_norm, _check_rotary, _norm_inputs, _qk, _rand, _replays, _within

pytestmark = pytest.mark.gpu


def test_rotary_axis_that_the_positions_do_not_hold():
    """A plan built by hand, of axes -1, 0, 1 and 2, with positions of two columns: pairs of axes 0 and 1 turn as they should,
    the others are NaN and not turned by another axis's position."""
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    for pairs in ("interleaved", "half"):
        freq = Rotary.build(32, DEV).freq
        axis = torch.tensor([0] * 5 + [1] * 5 + [2] * 5 + [-1], dtype=torch.int32, device=DEV)
        q, k = _qk(70, 2, 9, 3, 2, 40, "fp32")
        pos = torch.randint(0, 500, (2, 9, 2), device=DEV, generator=_rand(71))
        first = torch.arange(16, device=DEV)
        first, second = (2 * first, 2 * first + 1) if pairs == "interleaved" else (first, first + 16)
        held = torch.cat((first[:10], second[:10], torch.arange(32, 40, device=DEV)))
        for x, o in zip((q, k), rotary_embed(q, k, pos, Rotary(freq, axis, pairs))):
            want, mag = block.rotary(x, pos, freq, axis.clamp(0, 1), pairs)
            # (positions up to 500 of a frequency of 1: the 64-bit angle adds nothing to the 12 roundings)
            _within(o[..., held], (want[..., held], mag[..., held]), pairs, 13)
            assert bool(o[..., first[10:]].isnan().all()) and bool(o[..., second[10:]].isnan().all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 256), (5, 1001, 256), (3, 37, 300), (70, 4004, 392), (1030, 2320, 256),
                                   (1030, 2310, 256)])
def test_w4_linear_adds_an_fp32_bias_unrounded(m, n, k, dtype):
    """nn.Linear's own parameters are fp32. With a bias far larger than the products the output is the bias, rounded once:
    rounded to x's type first it would be off by up to a whole step where half of one is allowed."""
    from lingbot_world_v2_realtime_amd.layers.linear import W4Linear
    torch.manual_seed(m + n)
    lin = torch.nn.Linear(k, n).to(DEV)
    with torch.no_grad():
        lin.bias.normal_(std=30.0)
    for fmt, zeros in (("int4", True), ("fp4", False)):
        mod = W4Linear(lin, 64, fmt, zeros)
        sc, z = block.unpack_scale(mod.w4_scale), None if mod.w4_zero is None else block.unpack_scale(mod.w4_zero)
        value = block.w4_values(block.unpack_w4(mod.w4, fmt), sc, z, fmt)[:n, :k]
        x = torch.randn(m, k, device=DEV, generator=_rand(m)).to(DT[dtype])
        mag = x.double().abs() @ (sc.double().repeat_interleave(64, 1)[:n, :k] * 62).t().contiguous()
        want = x.double() @ value.t().contiguous() + lin.bias.double()
        with torch.no_grad():
            got = mod(x)
        assert got.dtype == x.dtype
        _within(got, (want, mag + want.abs()), f"{m}x{n}x{k} {fmt} {dtype}", k / 16 + 24)
        # a bias that records a gradient is added after the kernel: one more rounding, of the product alone
        y = mod(x)
        assert y.dtype == x.dtype
        half = torch.finfo(x.dtype).eps / 2
        err = (y.detach().double() - want).abs()
        tol = half * want.abs() + half * (want - lin.bias.double()).abs() + (k / 16 + 24) * 2.0 ** -24 * (mag + want.abs())
        assert bool((err <= 1.02 * tol).all())   # (a rounding of what a rounding gave: products of two halves, under 2^-8)
        (g,) = torch.autograd.grad(y, lin.bias, torch.ones_like(y))
        assert torch.equal(g, torch.full_like(lin.bias, m))


@pytest.mark.parametrize("m", [1, 40, 1030])
def test_gemm_w4_zeros_past_the_codes(m):
    """Zeros of any byte, as checkpoints that count them from one hold 16: the value is code - zero all the same."""
    from lingbot_world_v2_realtime_amd import kernels
    g, n, k = _rand(72), 2320, 256
    codes = torch.randint(0, 16, (n, k), device=DEV, generator=g, dtype=torch.uint8)
    scale = (torch.rand(n, 4, device=DEV, generator=g) + 0.1).bfloat16()
    zero = torch.randint(0, 256, (n, 4), device=DEV, generator=g, dtype=torch.uint8)
    zero[0] = 16
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    want = x.double() @ block.w4_values(codes, scale, zero, "int4").t().contiguous()
    # what the products and their offset add: codes up to 31 steps, zeros up to 255 + 16
    mag = x.double().abs() @ (scale.double().repeat_interleave(64, 1) * 302).t().contiguous()
    _within(kernels.gemm_w4(x, *kernels.pack_w4(codes, scale, zero.float())), (want, mag + want.abs()), f"{m} rows", k / 16 + 24)


# ---------------------------------------------------------------- the forms that a chunk's sizes take


# forward, more than 1024 rows: one wave a row with one, two and three pieces of 8 values a thread (up to 512, 1024 and
# 1536 channels), several waves with two and three, whole units and value by value
@pytest.mark.parametrize("c,dtype,vec", [(512, "fp16", "fp32"), (768, "bf16", "fp32"), (1536, "bf16", "fp32"),
                                         (1536, "fp16", "fp16"), (1536, "fp32", "fp32"), (771, "bf16", "bf16"),
                                         (1531, "fp16", "fp32"), (2048, "bf16", "bf16"), (4096, "fp16", "fp16"),
                                         (12288, "bf16", "fp32")])
def test_gated_norm_many_rows(c, dtype, vec):
    for norm, post, b, n, rows in (("layer", None, 1, 1100, 4), ("rms", "rms", 3, 371, 2), ("layer", "layer", 1, 1037, 5)):
        a = _norm_inputs(c + n, b, n, c, dtype, vec, norm, post, rows=rows)
        _check_norm(a, f"{b}x{n}x{c} {dtype}/{vec} {norm}/{post}", norm=norm, post_norm=post)


# backward with a norm on both sides and both outputs' gradients: every count of pieces a thread and of waves a row, few
# rows and a chunk's, of which a workgroup takes more than its least of four (bounds as in test_gpu_block.py: at most 8
# rows in a thread's turn and 900 workgroups' sums over 32 slices, far under 160 additions)
@pytest.mark.parametrize("norm,post", [("rms", "rms"), ("layer", "layer"), ("rms", "layer"), ("layer", "rms")])
@pytest.mark.parametrize("b,n,c,dtype,mod", [(1, 1500, 512, "bf16", "rows"), (1, 1500, 1024, "fp16", "shared"),
                                             (2, 777, 1536, "bf16", "rows"), (1, 300, 2048, "bf16", "rows"),
                                             (2, 259, 4096, "fp16", "shared"), (2, 70, 4090, "bf16", "rows"),
                                             (1, 66, 5120, "fp32", "shared"), (1, 37, 8192, "bf16", "rows"),
                                             (2, 19, 8200, "fp16", "shared"), (1, 41, 12288, "bf16", "rows"),
                                             (1, 13, 12285, "fp32", "rows"), (1, 6032, 1536, "bf16", "rows"),
                                             (1, 1100, 12288, "bf16", "shared"), (1, 4500, 2048, "fp16", "shared")])
def test_gated_norm_gradients_with_norms_on_both_sides(b, n, c, dtype, mod, norm, post):
    a = _norm_inputs(n + c, b, n, c, dtype, None, norm, post, mod, 4)
    g = _rand(c)
    ds, dh = (torch.randn(b, n, c, device=DEV, generator=g).to(DT[dtype]) for _ in range(2))
    _check_norm(a, f"{b}x{n}x{c} {dtype} {norm}/{post}/{mod}", ds, dh, norm=norm, post_norm=post)


# several tokens a workgroup (2, 4 and 8), the entries of a batch ending inside one, k beside q; units of 16 bytes, of 8
# and single values
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("b,n,hq,hk,d,rot,dtype", [(3, 1001, 12, 2, 128, 128, "bf16"), (3, 1001, 3, 1, 128, 64, "fp32"),
                                                   (3, 2749, 4, 4, 128, 64, "fp16"), (5, 3333, 1, 1, 64, 64, "bf16"),
                                                   (5, 3333, 2, 1, 96, 24, "fp16"), (7, 2347, 1, 0, 7, 6, "bf16"),
                                                   (3, 1001, 2, 2, 80, 70, "bf16")])
def test_rotary_several_tokens_a_workgroup(b, n, hq, hk, d, rot, dtype, pairs):
    from lingbot_world_v2_realtime_amd import Rotary
    q, k = _qk(n + d, b, n, hq, hk, d, dtype)
    rope = Rotary.build(rot, DEV, pairs=pairs)
    pos = torch.randint(0, 5000, (b, n), device=DEV, generator=_rand(2))
    _check_rotary(q, k, pos, rope, f"{dtype} {pairs} {b}x{n}x{hq}/{hk}x{d}/{rot}")
    _check_rotary(q.transpose(1, 2), None if k is None else k.transpose(1, 2), 77, rope, "HND, one position", "HND")


def test_rotary_three_axes_of_a_chunk():
    """A chunk's grid at its start frame, two entries of the batch at different ones."""
    from lingbot_world_v2_realtime_amd import Rotary, grid_positions
    rope = Rotary.build(128, DEV, sections=(22, 21, 21))
    q, k = _qk(73, 2, 4 * 29 * 13, 3, 1, 128)
    pos = torch.stack([grid_positions((4, 29, 13), f, DEV) for f in (0, 1000)])
    _check_rotary(q, k, pos, rope, "chunk")


def test_rotary_needs_a_head():
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    rope = Rotary.build(128, DEV)
    q, k = _qk(74, 1, 5, 4, 2, 128)
    for bad in ((q[:, :, :0], k), (q, k[:, :, :0])):
        with pytest.raises(ValueError, match="a head at least"):
            rotary_embed(*bad, 0, rope)
    oq, ok = rotary_embed(q[:, :, :0], k[:, :, :0], 0, rope)   # nothing at all is no error
    assert oq.numel() == ok.numel() == 0


# ---------------------------------------------------------------- calls in a graph, in place, from several threads


def test_module_and_inplace_rotation_in_a_graph():
    """A 4-bit linear with an fp32 bias and a rotation in place, captured together and replayed with other inputs; eager calls
    run between the replays."""
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    from lingbot_world_v2_realtime_amd.layers.linear import W4Linear
    torch.manual_seed(5)
    mod, rope = W4Linear(torch.nn.Linear(256, 6 * 128).to(DEV), 64, "int4", True), Rotary.build(128, DEV, pairs="half")
    x = torch.randn(9, 256, device=DEV, generator=_rand(75)).bfloat16()
    pos = torch.arange(9, device=DEV)

    def make():
        with torch.no_grad():
            y = mod(x).view(1, 9, 6, 128)
            rotary_embed(y[:, :, :4], y[:, :, 4:5], pos, rope, inplace=True)
        return [y]

    _replays(make, lambda i: (x.add_(0.25), pos.add_(3)))


def test_two_threads_on_two_streams():
    """Two host threads, each with a stream and inputs of its own, forward and backward, fifty calls each: every result is the
    bits of a call alone."""
    import threading

    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    rope, results = Rotary.build(128, DEV), {}

    def step(a, pos):
        s, h = gated_norm(**a)
        q, _ = rotary_embed(h.view(1, 90, 4, 128), None, pos, rope)
        return [s.detach(), q.detach(), *torch.autograd.grad((s, q), list(a.values()), (torch.ones_like(s), torch.ones_like(q)))]

    inputs = []
    for seed in (76, 77):
        a = {k: v.requires_grad_() for k, v in _norm_inputs(seed, 1, 90, 512, "bf16", "fp32").items()}
        pos = torch.randint(0, 9999, (90,), device=DEV, generator=_rand(seed))
        inputs.append((a, pos, [t.clone() for t in step(a, pos)]))
    torch.cuda.synchronize()

    def work(i):
        a, pos, want = inputs[i]
        stream, same = torch.cuda.Stream(), True
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = step(a, pos)
                same = same and all(torch.equal(x, y) for x, y in zip(got, want))
            stream.synchronize()
        results[i] = same

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert results == {0: True, 1: True}


@pytest.mark.parametrize("m", [1, 40, 1030])
@pytest.mark.parametrize("fmt,zeros", [("int4", False), ("int4", True), ("fp4", False)])
def test_gemm_w4_small_and_large_rows(m, fmt, zeros):
    """Rows below the format's normal numbers, rows near fp16's largest, and rows of one sign, whose codes' offset is far larger
    than what remains of it."""
    from lingbot_world_v2_realtime_amd import kernels
    n, k = 2320, 256
    for dtype, size, std in (("fp16", 2.0 ** -20, 200.0), ("bf16", 2.0 ** -130, 1.0), ("fp16", 3e4, 2.0 ** -12),
                             ("bf16", 2.0 ** 100, 1.0), ("bf16", 1.0, 1.0)):
        g = _rand(78)
        codes = torch.randint(0, 16, (n, k), device=DEV, generator=g, dtype=torch.uint8)
        scale = ((torch.rand(n, 4, device=DEV, generator=g) + 0.1) * std).bfloat16()
        zero = torch.randint(0, 16, (n, 4), device=DEV, generator=g, dtype=torch.uint8) if zeros else None
        x = (torch.rand(m, k, device=DEV, generator=g, dtype=torch.float64) * 0.9 + 0.1) * size
        if size != 1.0:
            x = x * (1 - 2 * torch.randint(0, 2, (m, k), device=DEV, generator=g))
        x = x.to(DT[dtype])
        want = x.double() @ block.w4_values(codes, scale, zero, fmt).t().contiguous()
        steps = 62 if fmt == "int4" else 6
        mag = x.double().abs() @ (scale.double().repeat_interleave(64, 1) * steps).t().contiguous()
        _within(kernels.gemm_w4(x, *kernels.pack_w4(codes, scale, zero, fmt), fmt=fmt), (want, mag + want.abs()),
                f"{m} rows of {dtype} around {size}", k / 16 + 24)


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
def test_rotary_fp32_values_keep_the_angle(pairs):
    """fp32 q: the factors are off by their functions' last bits (4 * 2^-24) and the rounding of what corrects the angle's (1),
    each product by another: 6 * 2^-24 of what is added, beside the sum's own (positions up to 5000: the 64-bit angle is good
    to 2e-12). On the whole no further off than the same products by torch with sine and cosine taken in 64 bits."""
    from lingbot_world_v2_realtime_amd import Rotary, rotary_embed
    q, _ = _qk(79, 1, 5000, 4, 0, 128, "fp32")
    rope, pos = Rotary.build(128, DEV, pairs=pairs), torch.arange(5000, device=DEV)
    want = block.rotary(q, pos, rope.freq, pairs=pairs)
    got = rotary_embed(q, None, pos, rope)[0]
    _within(got, want, pairs, 6)
    angle = pos.double()[:, None] * rope.freq
    cos, sin = angle.cos().float()[None, :, None], angle.sin().float()[None, :, None]
    a, b = (q[..., 0::2], q[..., 1::2]) if pairs == "interleaved" else (q[..., :64], q[..., 64:])
    parts = (a * cos - b * sin, b * cos + a * sin)
    plain = torch.stack(parts, -1).flatten(-2) if pairs == "interleaved" else torch.cat(parts, -1)
    rms = [(t.double() - want[0]).square().mean().sqrt().item() for t in (got, plain)]
    assert rms[0] <= rms[1], rms


# ---------------------------------------------------------------- gradients by halves


@pytest.mark.parametrize("shapes", [("rows", "shared", "none"), ("shared", "rows", "rows"), ("none", "rows", "shared"),
                                    ("rows", "none", "rows"), ("shared", "shared", "rows")])
def test_gated_norm_modulations_of_different_shapes(shapes):
    """gate, shift and scale each with rows of its own, shared or absent."""
    b, n, c, rows = 2, 61, 520, 4
    a = _norm_inputs(80, b, n, c, "bf16", "fp32", "layer", "rms", "rows", rows)
    for name, shape in zip(("gate", "shift", "scale"), shapes):
        if shape == "shared":
            a[name] = a[name][0, 1].clone()
        elif shape == "none":
            del a[name]
    g = _rand(81)
    ds, dh = (torch.randn(b, n, c, device=DEV, generator=g).bfloat16() for _ in range(2))
    kw = dict(post_norm="rms", group_len=17)
    _check_norm(a, f"{shapes}", ds, dh, **kw)


@pytest.mark.parametrize("branch", [False, True])
def test_gated_norm_each_gradient_alone(branch):
    """Only one input records a gradient, whichever others are there: the bits it has among all."""
    from lingbot_world_v2_realtime_amd import gated_norm
    a = _norm_inputs(82, 2, 37, 520, "fp16", "fp32", rows=3)
    if not branch:
        a = {k: v for k, v in a.items() if k not in ("y", "gate", "post_weight")}
    g = _rand(83)
    d = [torch.randn(2, 37, 520, device=DEV, generator=g).half() for _ in range(2 if branch else 1)]

    def grads(names):
        leaf = {k: v.detach().requires_grad_(k in names) for k, v in a.items()}
        out = gated_norm(**leaf)
        return dict(zip(names, torch.autograd.grad(out, [leaf[k] for k in names], d)))

    every = grads(list(a))
    for name in a:
        assert torch.equal(grads([name])[name], every[name]), name


def test_gradients_of_a_batch_of_gradients_are_refused():
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    x = torch.randn(1, 4, 64, device=DEV, requires_grad=True)
    rope = Rotary.build(64, DEV)
    for f in (lambda t: gated_norm(t), lambda t: rotary_embed(t.view(1, 4, 1, 64), None, 0, rope)[0]):
        y = f(x)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, x, torch.randn(3, *y.shape, device=DEV), is_grads_batched=True)


def test_gradients_by_saved_tensor_hooks_and_checkpoints():
    """Saved tensors moved to the host and back, and a forward run again by a checkpoint: the same bits."""
    from torch.utils.checkpoint import checkpoint

    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    a = {k: v.requires_grad_() for k, v in _norm_inputs(84, 1, 30, 512, "bf16", "fp32").items()}
    rope, pos = Rotary.build(128, DEV), torch.arange(30, device=DEV)

    def step(*ts):
        s, h = gated_norm(**dict(zip(a, ts)))
        return s, rotary_embed(h.view(1, 30, 4, 128), None, pos, rope)[0]

    def grads(out):
        return torch.autograd.grad(out, list(a.values()), [torch.ones_like(o) for o in out])

    want = grads(step(*a.values()))
    with torch.autograd.graph.save_on_cpu():
        got = step(*a.values())
    assert all(torch.equal(x, y) for x, y in zip(grads(got), want))
    assert all(torch.equal(x, y) for x, y in zip(grads(checkpoint(step, *a.values(), use_reentrant=False)), want))


def test_operators_in_a_compiled_function():
    """Inside torch.compile the calls are made as they are, between the compiled pieces."""
    from lingbot_world_v2_realtime_amd import Rotary, gated_norm, rotary_embed
    rope = Rotary.build(64, DEV)
    x = torch.randn(1, 6, 64, device=DEV, requires_grad=True)

    def f(t):
        h = gated_norm(t * 2, norm="rms") + 1
        return rotary_embed(h.view(1, 6, 1, 64), None, 3, rope)[0] * 0.5

    want = f(x)
    got = torch.compile(f, backend="eager")(x)
    assert torch.equal(got, want)
    assert torch.equal(torch.autograd.grad(got.sum(), x)[0], torch.autograd.grad(want.sum(), x)[0])


def test_a_gradient_without_memory_is_refused():
    """A hook that puts a stand-in for another tensor in a gradient's place: it must not count as no gradient."""
    from lingbot_world_v2_realtime_amd import gated_norm
    from test_block_calls import _StandIn
    x = torch.randn(1, 4, 64, device=DEV, requires_grad=True)
    s, h = gated_norm(x, x.detach())
    s.register_hook(_StandIn)
    with pytest.raises(RuntimeError, match="without memory"):
        torch.autograd.grad((s, h), x, (torch.ones_like(s), torch.ones_like(h)))
