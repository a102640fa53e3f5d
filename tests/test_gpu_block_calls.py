"""Calls that the block operators' documentation allows at the edges of their sizes, layouts and types, on the GPU against
the definitions in 64 bits (oracle/block.py), with the bounds of test_gpu_block.py."""
import pytest
import torch

from oracle import block
from test_gpu_block import DEV, DT, _qk, _rand, _within

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
