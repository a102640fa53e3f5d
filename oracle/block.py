"""The block operators in 64 bits: gated norm with its gradients, rotary positions, 4-bit weights. Each also gives, next
to a value, the magnitude that a 32-bit evaluation's rounding is relative to (what was added and multiplied on the way),
for error bounds.
"""
import torch

FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _unit(x, kind, eps, mag):
    """(unit, factor, magnitude of unit's error) of a row whose values carry errors relative to `mag`."""
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    d = x - mean
    r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = d * r
    # the row's largest error of a difference, times r, moves every value of the row through its statistics too
    worst = (mag + mag.mean(-1, keepdim=True)).amax(-1, keepdim=True) * r
    return u, r, worst * (1 + u.abs())


def gated_norm(x, y=None, gate=None, shift=None, scale=None, weight=None, bias=None, post_weight=None, norm="layer",
               post_norm=None, eps=1e-6, residual_scale=1.0, branch_scale=1.0, group_len=None, ds=None, dh=None):
    """((s, |s|), (h, |h|), grads) in float64; grads: name -> (value, magnitude), where ds or dh is given."""
    t = {"x": x, "y": y, "gate": gate, "shift": shift, "scale": scale, "weight": weight, "bias": bias,
         "post_weight": post_weight}
    t = {k: v.detach().double() for k, v in t.items() if v is not None}
    b, n, c = x.shape
    rows = next((v.shape[1] for v in (gate, shift, scale) if v is not None and v.dim() == 3), 1)
    group_len = group_len or max(-(-n // rows), 1)
    row = torch.arange(n, device=x.device) // group_len

    def tok(name, other):
        v = t.get(name)
        return torch.full((c,), float(other), dtype=torch.float64, device=x.device) if v is None else \
            v if v.dim() == 1 else v[:, row]

    al, be = residual_scale, branch_scale
    gp = be * tok("gate", 1) * tok("post_weight", 1)
    s, s_mag = al * t["x"], (al * t["x"]).abs()
    v = v_mag = rv = None
    if y is not None:
        if post_norm is None:
            v, v_mag = t["y"], t["y"].abs()
        else:
            v, rv, v_mag = _unit(t["y"], post_norm, eps, t["y"].abs())
        s, s_mag = s + gp * v, s_mag + gp.abs() * v_mag
    h = h_mag = None
    w, cc, m = tok("weight", 1), tok("bias", 0), 1 + tok("scale", 0)
    if norm is not None:
        u, r, u_mag = _unit(s, norm, eps, s_mag)
        lin, lin_mag = u * w + cc, u_mag * w.abs() + cc.abs()
        h = lin * m + tok("shift", 0)
        h_mag = lin_mag * (1 + tok("scale", 0).abs()) + tok("shift", 0).abs()
    if ds is None and dh is None:
        return (s, s_mag), (h, h_mag), {}

    def through(d, d_mag, unit, unit_mag, r, kind):
        """The gradient through unit = (x - mean) r, and its magnitude."""
        k = (d * unit).mean(-1, keepdim=True)
        k_mag = (d_mag * (unit.abs() + unit_mag)).mean(-1, keepdim=True)
        out = d - unit * k
        mag = d_mag + (unit.abs() + unit_mag) * k_mag
        if kind == "layer":
            out = out - d.mean(-1, keepdim=True)
            mag = mag + d_mag.mean(-1, keepdim=True)
        return out * r, mag * r * (1 + unit_mag.amax(-1, keepdim=True))

    g = torch.zeros_like(s) if ds is None else ds.double()
    g_mag = g.abs()
    each = {}
    if dh is not None:
        d = dh.double()
        du, du_mag = d * m * w, d.abs() * (1 + tok("scale", 0).abs()) * w.abs()
        a, a_mag = through(du, du_mag, u, u_mag, r, norm)
        g, g_mag = g + a, g_mag + a_mag
        each.update(shift=(d, d.abs()), scale=(d * lin, d.abs() * lin_mag), bias=(d * m, d.abs() * (1 + tok("scale", 0).abs())),
                    weight=(d * m * u, d.abs() * (1 + tok("scale", 0).abs()) * u_mag))
    grads = {"x": (al * g, abs(al) * g_mag)}
    if y is not None:
        dv, dv_mag = g * gp, g_mag * gp.abs()
        grads["y"] = (dv, dv_mag) if post_norm is None else through(dv, dv_mag, v, v_mag, rv, post_norm)
        pw, gt = tok("post_weight", 1), tok("gate", 1)
        each["gate"] = (be * g * pw * v, abs(be) * g_mag * pw.abs() * v_mag)
        each["post_weight"] = (be * g * gt * v, abs(be) * g_mag * gt.abs() * v_mag)
    for name, val in t.items():
        if name in ("x", "y"):
            continue
        out = []
        for part in each.get(name, (torch.zeros_like(s),) * 2):
            if val.dim() == 1:
                out.append(part.sum((0, 1)))
            else:
                z = torch.zeros(val.shape, dtype=torch.float64, device=x.device)
                out.append(z.index_add_(1, row, part))
        grads[name] = tuple(out)
    return (s, s_mag), (h, h_mag), {k: v for k, v in grads.items() if k in t}


def rotary(x, positions, freq, axis=None, pairs="interleaved", factor=1.0, inverse=False):
    """(value, magnitude) of x [B, L, H, D] rotated; positions [B, L] or [L], with an axis array [.., axes]."""
    x = x.detach().double()
    b, n = x.shape[:2]
    p = positions.double()
    if axis is None:
        ang = p[..., None] * freq
    else:
        ang = p[..., axis.long()] * freq
    ang = ang.expand(b, n, -1)[:, :, None] * (-1 if inverse else 1)
    k = freq.shape[0]
    i = torch.arange(k, device=x.device)
    i0, i1 = (2 * i, 2 * i + 1) if pairs == "interleaved" else (i, i + k)
    out, mag = x.clone(), torch.zeros_like(x)
    c, s = factor * ang.cos(), factor * ang.sin()
    out[..., i0] = x[..., i0] * c - x[..., i1] * s
    out[..., i1] = x[..., i1] * c + x[..., i0] * s
    mag[..., i0] = mag[..., i1] = abs(factor) * (x[..., i0].abs() + x[..., i1].abs())
    return out, mag


def unpack_w4(w4, fmt):
    """Tiles [N/16, K/128, 1024] -> codes uint8 [N, K], word by word from the layout's definition."""
    nt, kt, _ = w4.shape
    words = w4.reshape(nt, kt, 64, 4, 4).to(torch.int64)
    words = words[..., 0] | words[..., 1] << 8 | words[..., 2] << 16 | words[..., 3] << 24   # [nt, kt, lane, word]
    out = torch.zeros(nt, 16, kt, 128, dtype=torch.uint8, device=w4.device)
    for q in range(4):
        for j in range(4):
            for s in range(8):
                i = s if fmt == "fp4" else (2 * s if s < 4 else 2 * s - 7)
                out[:, :, :, 32 * j + 8 * q + i] = \
                    (words[:, :, 16 * q:16 * q + 16, j] >> 4 * s & 15).to(torch.uint8).transpose(1, 2)
    return out.reshape(nt * 16, kt * 128)


def unpack_scale(scale):
    """[N/16, K/128, 16, groups] -> [N, K / group]."""
    nt, kt, _, g = scale.shape
    return scale.transpose(1, 2).reshape(nt * 16, kt * g)


def w4_values(codes, scale, zero, fmt):
    """Weights [N, K] in float64 of codes [N, K] and scales, zeros [N, K / group]."""
    g = codes.shape[1] // scale.shape[1]
    if fmt == "fp4":
        v = FP4.to(codes.device)[(codes & 7).long()] * (1 - 2 * (codes >> 3).double())
    else:
        v = codes.double() - (8.0 if zero is None else zero.double().repeat_interleave(g, 1))
    return v * scale.double().repeat_interleave(g, 1)


def quant_w4(w, group, fmt, zeros=False):
    """(codes, scale bf16, zero or None) of a float32 weight [N, K], K a multiple of `group`: the formula in 32 bits."""
    n, k = w.shape
    v = w.float().reshape(n, k // group, group)
    hi, lo = v.amax(2, keepdim=True).clamp(min=0), v.amin(2, keepdim=True).clamp(max=0)
    amax = torch.maximum(hi, -lo)
    scale = (amax / 6 if fmt == "fp4" else (hi - lo) / 15 if zeros else amax / 7).to(torch.bfloat16)
    s = scale.float()
    s = torch.where(s >= 2.0 ** -126, s, torch.zeros_like(s))
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    zero = None
    if fmt == "fp4":
        u = torch.where(s > 0, v / s, torch.zeros_like(v))
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
        codes = torch.bucketize(u.abs(), mids) + 8 * (u < 0)
    else:
        z = (-lo * inv).round().clamp(0, 15) if zeros else torch.full_like(lo, 8.0)
        codes = (v * inv + z).round().clamp(0, 15)
        zero = z[:, :, 0].to(torch.uint8) if zeros else None
    return codes.to(torch.uint8).reshape(n, k), s[:, :, 0].to(torch.bfloat16), zero


def w4_linear(x, w, bias=None):
    """(value, magnitude) of x w^T + bias; the magnitude counts the integer codes' offset (31 + 8 steps of a scale at
    most where a weight is a step or more: bounded by 40 |w| + the group's scale, taken by the caller's bound)."""
    x, w = x.double(), w.double()
    y, mag = x @ w.t().contiguous(), x.abs() @ w.abs().t().contiguous()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag
