"""Calls of the block operators that have no right answer, on the CPU: each is refused, and says why, before anything
looks for a device."""
import pytest
import torch
from torch.autograd import forward_ad

from lingbot_world_v2_realtime_amd import _lib, kernels
from lingbot_world_v2_realtime_amd.layers.linear import W4Linear, convert_to_w4
from lingbot_world_v2_realtime_amd.layers.norm import gated_norm
from lingbot_world_v2_realtime_amd.layers.rotary import Rotary, rotary_embed
from oracle import block


@pytest.fixture
def w4_module(monkeypatch):
    """A W4Linear of 1536 -> 32 with empty tiles (the quantisation itself needs the GPU)."""
    def tiles(w, group, fmt, zeros):
        shapes = kernels._w4_shapes(*w.shape, group)
        return torch.zeros(shapes[0], dtype=torch.uint8), torch.zeros(shapes[1], dtype=torch.bfloat16), None
    monkeypatch.setattr(kernels, "quant_w4", tiles)
    return W4Linear(torch.nn.Linear(1536, 32))


@pytest.mark.parametrize("width", [1500, 1409, 1535, 1408, 1537, 1])
def test_w4_linear_refuses_another_width(w4_module, width):
    """1409 to 1535 columns end in the weights' last tile of 128: the tiles alone do not tell them from 1536."""
    with torch.no_grad(), pytest.raises(ValueError, match=f"1536 .*{width}"):
        w4_module(torch.zeros(2, width, dtype=torch.bfloat16))


def _recording(t, how):
    if how == "gradient":
        return t.clone().requires_grad_()
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("how", ["gradient", "tangent"])
def test_raw_calls_do_not_lose_a_gradient(how):
    """The functions of kernels.py that have no gradient of their own refuse a call that would record one, whichever tensor
    asks for it: their results would be detached without a word."""
    x = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    norm = dict(x=x, y=x.clone(), gate=x[0, 0].clone(), weight=x[0, 0].clone())
    q = x.view(1, 4, 1, 128)
    freq = torch.ones(8, dtype=torch.float64)
    gemm = dict(x=x[0], w4=torch.zeros(1, 1, 1024, dtype=torch.uint8), scale=torch.zeros(1, 1, 16, 1, dtype=torch.bfloat16),
                bias=torch.zeros(16, dtype=torch.bfloat16))
    with forward_ad.dual_level():
        for name in ("x", "bias", "scale"):
            with pytest.raises(RuntimeError, match="gemm_w4.*gradient"):
                kernels.gemm_w4(**{**gemm, name: _recording(gemm[name], how)})
        for name in norm:
            args = {**norm, name: _recording(norm[name], how)}
            with pytest.raises(RuntimeError, match="gated_norm.*gradient"):
                kernels.gated_norm(**args)
            with pytest.raises(RuntimeError, match="gated_norm_bwd.*gradient"):
                kernels.gated_norm_bwd(args.pop("x"), x, x, **args)
        with pytest.raises(RuntimeError, match="gated_norm_bwd.*gradient"):
            kernels.gated_norm_bwd(x, _recording(x, how), x)
        for args in (dict(q=_recording(q, how), k=None), dict(q=q, k=_recording(q, how)),
                     dict(q=q, k=None, q_out=_recording(q, how))):
            with pytest.raises(RuntimeError, match="rotary.*gradient"):
                kernels.rotary(**args, positions=0, freq=freq)


def test_raw_calls_without_grad_mode_go_on():
    """As the forward of a user's own autograd function has them: what is refused then is the host tensor."""
    x = torch.zeros(1, 4, 128, dtype=torch.bfloat16, requires_grad=True)
    with torch.no_grad():
        for call in (lambda: kernels.gated_norm(x), lambda: kernels.gated_norm_bwd(x, None, x),
                     lambda: kernels.rotary(x.view(1, 4, 1, 128), None, 0, torch.ones(8, dtype=torch.float64)),
                     lambda: kernels.gemm_w4(x[0], torch.zeros(1, 1, 1024, dtype=torch.uint8),
                                             torch.zeros(1, 1, 16, 1, dtype=torch.bfloat16))):
            with pytest.raises(ValueError, match="device tensor"):
                call()


@pytest.mark.parametrize("axes", [1, 2])
@pytest.mark.parametrize("batch", [False, True])
def test_rotary_positions_need_every_axis_of_the_plan(axes, batch):
    """A plan of frame, row and column with positions of two columns (or one) has nothing to turn the last section by."""
    rope = Rotary.build(128, "cpu", sections=(22, 21, 21))
    q = torch.zeros(2, 6, 1, 128, dtype=torch.bfloat16)
    pos = torch.zeros((2, 6, axes) if batch else (6, axes), dtype=torch.int64)
    assert rope.axes == 3 and Rotary.build(128, "cpu").axes == 1
    with pytest.raises(ValueError, match="3 axes"):
        rotary_embed(q, None, pos, rope)
    with pytest.raises(ValueError, match="3 axes"):
        kernels.rotary(q, None, pos, rope.freq, rope.axis, axes=rope.axes)


def test_a_plan_built_by_hand_may_leave_its_axes_open():
    rope = Rotary.build(128, "cpu", sections=(22, 21, 21))
    by_hand = Rotary(rope.freq, rope.axis, rope.pairs, rope.factor)
    assert by_hand.axes is None
    with pytest.raises(ValueError, match="axes"):
        rotary_embed(torch.zeros(1, 6, 1, 128), None, torch.zeros(6, 3, dtype=torch.int64), Rotary(rope.freq, rope.axis, axes=0))


def _answer(call):
    """'ok' where only the host tensors are refused, else what the call said."""
    with pytest.raises(ValueError) as e:
        call()
    said = str(e.value)
    return "ok" if "device tensor" in said else said


def _addresses(t):
    at = torch.tensor(t.storage_offset())
    for n, s in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * s
    return at.flatten().tolist()


FREQ = torch.ones(1, dtype=torch.float64)


def test_rotary_outputs_that_share_memory_are_refused():
    """Views with gaps, of which the channels, heads or tokens of one lie in the other: their threads would write over what
    others read. Views that only lie between each other are taken."""
    fused = torch.zeros(2, 5, 10, 8, dtype=torch.bfloat16)
    rope = Rotary(FREQ)

    def inplace(q, k=None):
        return _answer(lambda: rotary_embed(q, k, 0, rope, inplace=True))

    assert inplace(fused[:, :, :6], fused[:, :, 6:8]) == "ok"                 # q and k of one projection
    assert inplace(fused[:, :, ::2], fused[:, :, 1::2]) == "ok"               # alternating heads
    assert inplace(fused[:, :3], fused[:, 2:][:, :3]) != "ok"                 # a token of both
    assert inplace(fused[:, :, :6], fused[:, :, 5:7]) != "ok"                 # a head of both
    assert inplace(fused[..., :4], fused[..., 3:7]) != "ok"                   # a channel of both
    assert inplace(fused[..., :4], fused[..., 4:]) == "ok"
    flat = torch.zeros(400, dtype=torch.bfloat16)
    assert inplace(flat.as_strided((1, 20, 1, 8), (400, 8, 8, 1))) == "ok"
    assert "share" in inplace(flat.as_strided((1, 20, 1, 8), (400, 7, 8, 1)))      # windows one channel into the next
    assert "share" in inplace(flat.as_strided((2, 5, 3, 8), (40, 8, 40, 1)))       # two ways to the same head
    assert inplace(flat.as_strided((2, 3, 5, 8), (120, 40, 8, 1)).transpose(1, 2)) == "ok"

    def out(q, q_out, **kw):
        return _answer(lambda: kernels.rotary(q, None, 0, FREQ, q_out=q_out, **kw))

    assert out(fused[:, :, :6], fused[:, :, :6]) == "ok"                      # the input itself
    assert "overlaps" in out(fused[:, :, :6], fused[:, :, 1:7])
    assert "overlaps" in out(fused[..., :4], fused[..., 2:6])
    assert out(fused[:, :, :4], fused[:, :, 4:8]) == "ok"
    assert "overlaps" in out(fused[:, :2], fused[:, :2].transpose(0, 1))      # its memory in another order
    assert "share" in out(fused[:, :, :1], flat.as_strided((2, 5, 1, 8), (35, 7, 7, 1)))


@pytest.mark.parametrize("seed", range(4))
def test_rotary_overlaps_against_every_address(seed):
    """Two strided views of one buffer, of random sizes and steps, against the sets of their elements' addresses."""
    g = torch.Generator().manual_seed(seed)
    rope, seen = Rotary(FREQ), set()

    def draw(*of):
        return of[int(torch.randint(len(of), (), generator=g))]

    buf = torch.zeros(4096)
    for _ in range(300):
        b, n, h = draw(1, 2), draw(1, 2, 3), draw(1, 2, 3)
        d = draw(2, 3, 4)
        shape = (b, n, h, d)
        q, k = (buf.as_strided(shape, (draw(0, 5, 12, 24, 36, 72), draw(3, 4, 12, 13, 24), draw(2, 3, 4, 6, 8, 24), 1),
                               draw(0, 1, 2, 4, 6, 12, 16, 40, 100)) for _ in range(2))
        at = [_addresses(t) for t in (q, k)]
        own = [len(set(a)) == len(a) for a in at]
        apart = not set(at[0]) & set(at[1])
        same = at[0] == at[1]
        said = _answer(lambda: rotary_embed(q, k, 0, rope, inplace=True))
        assert (said == "ok") == (all(own) and apart), (shape, q.stride(), k.stride(), said)
        said = _answer(lambda: kernels.rotary(q, None, 0, FREQ, q_out=k))
        assert (said == "ok") == (own[1] and (apart or same)), (shape, q.stride(), k.stride(), said)
        seen.add((all(own), apart, same))
    assert len(seen) >= 4


def test_gemm_w4_takes_a_bias_of_its_own_type_only():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    tiles = torch.zeros(1, 1, 1024, dtype=torch.uint8), torch.zeros(1, 1, 16, 1, dtype=torch.bfloat16)
    for bias in (torch.zeros(16), torch.zeros(16, dtype=torch.float16)):
        with pytest.raises(ValueError, match="bias must be"):
            kernels.gemm_w4(x, *tiles, bias=bias)


def test_w4_entry_point_takes_an_fp32_bias():
    """Its flag beside the format: alignment of four bytes, and no other bit."""
    def gemm(dtype, bias):
        return _lib.load().lbw_gemm_w4(1 << 20, dtype, 3, 100, 100, 1 << 20, 1 << 20, None, 0, 64, 30, bias, 1 << 20, None)
    assert gemm(0, (1 << 20) + 1) == 3 and gemm(256, (1 << 20) + 2) == 3
    assert gemm(2, None) == 2 and gemm(256 + 2, None) == 2 and gemm(512, None) == 2


def test_pack_w4_refuses_what_its_bytes_cannot_hold():
    """Zeros that a cast to a byte would change, and codes of more than four bits, which would lose their upper ones."""
    codes, scale = torch.zeros(4, 128, dtype=torch.uint8), torch.ones(4, 2)
    for bad in (7.5, -1.0, 256.0, float("nan"), float("inf")):
        zero = torch.full((4, 2), 8.0)
        zero[3, 1] = bad
        with pytest.raises(ValueError, match="zeros must be whole numbers"):
            kernels.pack_w4(codes, scale, zero)
    for bad in (torch.full((4, 2), -1, dtype=torch.int8), torch.full((4, 2), 300)):
        with pytest.raises(ValueError, match="zeros must be whole numbers"):
            kernels.pack_w4(codes, scale, bad)
    for kind in (torch.float32, torch.float16, torch.int8, torch.int64, torch.uint8):
        z = kernels.pack_w4(codes, scale, torch.full((4, 2), 9, dtype=kind))[2]
        assert z.dtype == torch.uint8 and bool((block.unpack_scale(z)[:4, :2] == 9).all())
    codes[2, 77] = 16
    with pytest.raises(ValueError, match="0 .. 15"):
        kernels.pack_w4(codes, scale)


def test_gated_norm_bwd_names_its_gradients():
    """wants holds names of inputs: a plain string would be searched letter by letter (and 'weight' be found in
    'post_weight'), an unknown name would ask for nothing."""
    x = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    for bad in ("post_weight", "x", ("gat",), ("x", "wieght"), (0,)):
        with pytest.raises((ValueError, TypeError), match="wants"):
            kernels.gated_norm_bwd(x, None, x, wants=bad)
    for good in ((), ["x"], ("x", "gate"), {"x"}):
        with pytest.raises(ValueError, match="device tensor"):
            kernels.gated_norm_bwd(x, None, x, wants=good)


def test_w4_linear_says_what_it_cannot_take(w4_module):
    """A gradient, a tangent, a transform's stand-in and a tensor subclass are four reasons, not one."""
    class Marked(torch.Tensor):
        pass

    x = torch.zeros(2, 1536, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradient"):
        w4_module(x.clone().requires_grad_())
    with torch.no_grad():
        with pytest.raises(TypeError, match="Marked"):
            w4_module(x.as_subclass(Marked))
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.vmap(w4_module)(x[None])
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
            w4_module(forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(TypeError, match="tensor"):
        w4_module([1.0] * 1536)


def test_quant_w4_refuses_a_lazy_negation():
    """It is not in memory yet, and would be read without its sign."""
    with pytest.raises(ValueError, match="negated"):
        kernels.quant_w4(torch._neg_view(torch.ones(16, 128)))


def test_w4_linear_refuses_weights_that_are_not_finite(monkeypatch):
    """A NaN would become an ordinary code."""
    monkeypatch.setattr(kernels, "quant_w4", lambda *a: (torch.zeros(1, dtype=torch.uint8), torch.zeros(1), None))
    for bad in (float("nan"), float("inf")):
        lin = torch.nn.Linear(128, 16)
        with torch.no_grad():
            lin.weight[3, 5] = bad
        with pytest.raises(ValueError, match="finite"):
            W4Linear(lin)
        net = torch.nn.Sequential(torch.nn.Linear(128, 16), lin)
        with pytest.raises(ValueError, match="finite"):
            convert_to_w4(net, min_features=16)
        assert type(net[0]) is torch.nn.Linear   # nothing is replaced by a conversion that fails
    W4Linear(torch.nn.Linear(128, 16))


class _StandIn(torch.Tensor):
    """A tensor that stands for another and has no memory of its own, as distributed tensors do."""
    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device, strides=t.stride())

    def __init__(self, t):
        pass

    @classmethod
    def __torch_dispatch__(cls, *a, **kw):
        raise AssertionError("the operators look at tensors only")


def test_tensors_without_memory_are_refused():
    """An address of zero means 'absent' to the kernels: a weight, a branch or positions held by such a tensor would be left
    out of the result."""
    x = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    v, freq = x[0, 0].clone(), torch.ones(8, dtype=torch.float64)
    args = dict(x=x, y=x.clone(), gate=v, shift=v, scale=v, weight=v, bias=v, post_weight=v, post_norm="rms")
    for name in ("x", "y", "gate", "shift", "scale", "weight", "bias", "post_weight"):
        with pytest.raises(TypeError, match=f"^{name} has no memory"):
            gated_norm(**{**args, name: _StandIn(args[name])})
    q, axis = x.view(1, 4, 1, 128), torch.zeros(8, dtype=torch.int32)
    rotary = dict(q=q, k=q.clone(), positions=torch.zeros(4, 1, dtype=torch.int64), freq=freq, axis=axis)
    for name in rotary:
        with pytest.raises(TypeError, match=f"^{name} has no memory"):
            kernels.rotary(**{**rotary, name: _StandIn(rotary[name])})
    gemm = dict(x=x[0], w4=torch.zeros(1, 1, 1024, dtype=torch.uint8), scale=torch.zeros(1, 1, 16, 1, dtype=torch.bfloat16),
                zero=torch.zeros(1, 1, 16, 1, dtype=torch.uint8), bias=torch.zeros(16, dtype=torch.bfloat16))
    for name in gemm:
        with pytest.raises(TypeError, match=f"^{name} has no memory"):
            kernels.gemm_w4(**{**gemm, name: _StandIn(gemm[name])})
    with pytest.raises(ValueError, match="device tensor"):   # nothing to hold needs no memory
        gated_norm(torch.zeros(1, 0, 128))


@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_rotary_views_of_a_whole_projection_are_told_apart(layout):
    """q and k of a chunk's fused projection, in place: thousands of tokens whose addresses interleave, and no element of
    both; and the same with one head of both."""
    fused = torch.zeros(2, 6032, 36, 128, dtype=torch.bfloat16)
    if layout == "HND":
        fused = fused.transpose(1, 2)
    axis, rope = (2 if layout == "NHD" else 1), Rotary(torch.ones(64, dtype=torch.float64))
    view = lambda start, heads: fused.narrow(axis, start, heads)   # noqa: E731

    def inplace(q, k):
        return _answer(lambda: rotary_embed(q, k, 0, rope, layout, inplace=True))

    assert inplace(view(0, 12), view(12, 12)) == "ok"
    assert inplace(view(0, 12), view(24, 2)) == "ok"
    assert "share" in inplace(view(0, 12), view(11, 2))
    halves = fused.unflatten(axis, (18, 2)).movedim(axis + 1, 0)   # heads in turn
    assert inplace(halves[0], halves[1]) == "ok"


def test_rotary_token_steps_without_a_common_factor():
    flat = torch.zeros(4000000, dtype=torch.bfloat16)
    a = flat.as_strided((1, 6032, 1, 128), (0, 300, 0, 1))
    rope = Rotary(torch.ones(64, dtype=torch.float64))
    for start, shares in ((150, True), (300 * 6031 + 128, False)):
        b = flat.as_strided((1, 3000, 1, 128), (0, 701, 0, 1), start)
        said = _answer(lambda: rotary_embed(a[:, :3000], b, 0, rope, inplace=True))
        assert ("share" in said) == shares
