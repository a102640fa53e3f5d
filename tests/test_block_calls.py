"""Calls of the block operators that have no right answer, on the CPU: each is refused, and says why, before anything
looks for a device."""
import pytest
import torch
from torch.autograd import forward_ad

from lingbot_world_v2_realtime_amd import kernels
from lingbot_world_v2_realtime_amd.layers.linear import W4Linear
from lingbot_world_v2_realtime_amd.layers.rotary import Rotary, rotary_embed


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
