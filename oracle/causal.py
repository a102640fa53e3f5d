"""Causal self-attention in 64 bits: norms of q and k by head with the rotation, attention over packed sequences with its
gradients, and the cache in 4 bits. Next to a value stand the magnitudes that bounds of a 16- or 32-bit evaluation's error
are made of.
"""
import torch

from . import block


def norm_rotary(x, weight, positions, freq, axis=None, pairs="interleaved", factor=1.0, eps=1e-6, d=None):
    """((value, magnitude), grads) of x [B, L, H, D]; grads: 'x' and 'weight' -> (value, magnitude), from the output's d."""
    x = x.detach().double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.detach().double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    u = x * r
    y, mag = block.rotary(u * w, positions, freq, axis, pairs, factor)
    mag = torch.maximum(mag, (u * w).abs())   # (channels past the pairs)
    if d is None:
        return (y, mag), {}
    g, g_mag = block.rotary(d, positions, freq, axis, pairs, factor, inverse=True)
    g_mag = torch.maximum(g_mag, g.abs())
    grads = {"weight": ((g * u).sum((0, 1, 2)), (g_mag * u.abs()).sum((0, 1, 2)))}
    g, g_mag = g * w, g_mag * w.abs()
    k, k_mag = (g * u).mean(-1, keepdim=True), (g_mag * u.abs()).mean(-1, keepdim=True)
    grads["x"] = (r * (g - u * k), r * (g_mag + u.abs() * k_mag))
    return (y, mag), grads


def visible(n, m, causal, device):
    """[n, m]: whether query i sees key j, the last query being at the last key."""
    see = torch.ones(n, m, dtype=torch.bool, device=device)
    return see.tril(m - n) if causal else see


def attend(q, k, v, see, scale, d_out=None):
    """One sequence and head in float64: q [n, D] over k, v [m, D], see [n, m]. A dict: out, and of the bounds' parts: p_v = sum p
    |v|, p2_v2 = sum p^2 v^2, logit = the largest scale * sum |q| |k| of a row; with d_out also dq, dk, dv and for each of
    them `_abs` (sum of the magnitudes of what is added), `_sq` (sum of its squares), `_wide` (what errors of P, dP and D
    can move, for a relative error of 1 of each)."""
    q, k, v = q.double(), k.double(), v.double()
    s = q @ k.t().contiguous() * scale
    s = s.masked_fill(~see, float("-inf"))
    some = see.any(1, keepdim=True) if see.shape[1] else torch.zeros(q.shape[0], 1, dtype=torch.bool, device=q.device)
    top = s.amax(1, keepdim=True) if s.shape[1] else torch.zeros(q.shape[0], 1, dtype=torch.float64, device=q.device)
    e = torch.exp(s - torch.where(some, top, torch.zeros_like(top)))
    p = e / torch.where(some, e.sum(1, keepdim=True), torch.ones_like(top))
    r = {"out": p @ v, "p_v": p @ v.abs(), "p2_v2": p.square() @ v.square()}
    a = q.abs() @ k.abs().t().contiguous() * scale
    r["logit"] = a.masked_fill(~see, 0).amax(1, keepdim=True) if a.shape[1] else torch.zeros_like(top)
    if d_out is None:
        return r
    d = d_out.double()
    dp = d @ v.t().contiguous()
    delta = (d * r["out"]).sum(1, keepdim=True)
    ds = p * (dp - delta)
    r["dq"], r["dk"], r["dv"] = scale * ds @ k, scale * ds.t().contiguous() @ q, p.t().contiguous() @ d
    k_most = k.abs().amax(0, keepdim=True) if k.shape[0] else k.abs().sum(0, keepdim=True)
    r["dq_abs"] = scale * (ds.abs() @ k.abs() + ds.abs().sum(1, keepdim=True) * k_most)
    r["dk_abs"], r["dv_abs"] = scale * ds.abs().t().contiguous() @ q.abs(), p.t().contiguous() @ d.abs()
    r["dq_sq"] = scale ** 2 * ds.square() @ k.square()
    r["dk_sq"], r["dv_sq"] = scale ** 2 * ds.square().t().contiguous() @ q.square(), p.square().t().contiguous() @ d.square()
    # P's relative error moves P (dP - D) and D itself; dP and D have the error of their sums
    sums = d.abs() @ v.abs().t().contiguous() + (d.abs() * r["p_v"]).sum(1, keepdim=True)
    w16 = p * (p * dp.abs()).sum(1, keepdim=True)                                        # D from rounded P
    w32 = p * (sums + dp.abs() + delta.abs())
    for name, w in (("16", w16), ("32", w32)):
        r["dq_wide" + name] = scale * (w @ k.abs() + w.sum(1, keepdim=True) * k_most)
        r["dk_wide" + name] = scale * w.t().contiguous() @ q.abs()
    r["dv_wide16"], r["dv_wide32"] = torch.zeros_like(v), r["dv_abs"]
    r["dq_d2"] = scale ** 2 * (p.square() * (p.square() * dp.square()).sum(1, keepdim=True)) @ k.square()
    r["dk_d2"] = scale ** 2 * (p.square() * (p.square() * dp.square()).sum(1, keepdim=True)).t().contiguous() @ q.square()
    return r


def packed(q, k, v, starts, k_starts, scale=None, causal=True, d_out=None):
    """attend() of every sequence and head of packed rows: a dict of tensors like q (out, dq, ...) or k (dk, dv, ...; the sum over
    the heads that share one)."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    like = {}

    def put(name, ref, rows, head, x):
        if name not in like:
            like[name] = torch.zeros(*ref.shape[:2], x.shape[-1], dtype=torch.float64, device=ref.device)
        like[name][rows, head] += x

    for s in range(len(starts) - 1):
        rows, keys = slice(starts[s], starts[s + 1]), slice(k_starts[s], k_starts[s + 1])
        see = visible(starts[s + 1] - starts[s], k_starts[s + 1] - k_starts[s], causal, q.device)
        for h in range(q.shape[1]):
            r = attend(q[rows, h], k[keys, h // group], v[keys, h // group], see, scale, None if d_out is None else d_out[rows, h])
            for name, x in r.items():
                of_k = name[:2] in ("dk", "dv")
                put(name, k if of_k else q, keys if of_k else rows, h // group if of_k else h, x)
    return like


# ---------------------------------------------------------------- the cache

FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e, exactly (a device's pow need not be)."""
    table = torch.tensor([2.0 ** i for i in range(-200, 201)], dtype=torch.float64, device=e.device)
    return table[e.long() + 200]


def encode(x):
    """(codes, scales) int64 of x [..., D]: by the definition, value by value from the sixteen that there are."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(g).all(-1, keepdim=True)
    e = torch.full_like(top, 126.0)
    for s in range(126, -126, -1):
        e = torch.where(top <= 6 * 2.0 ** s, float(s), e)
    u = torch.where(fine, g, torch.zeros_like(g)).clamp(-3 * 2.0 ** 126, 3 * 2.0 ** 126) / _power(e)
    grid = torch.tensor(FP4, dtype=torch.float64, device=x.device)
    away = (u.abs()[..., None] - grid).abs()
    near = away.amin(-1, keepdim=True)
    # of two that are as near the even code
    rank = torch.where(away == near, torch.arange(8, device=x.device) % 2, 2)
    code = rank.argmin(-1) + 8 * torch.signbit(u).long()
    return code.flatten(-2), torch.where(fine, e + 127, torch.full_like(e, 255.0)).squeeze(-1).long()


def values(codes, scale):
    """float64 values of codes [..., D] with scales [..., D / 32]; scale 255: NaN."""
    grid = torch.tensor(FP4 + tuple(-v for v in FP4), dtype=torch.float64, device=codes.device)
    v = grid[codes.long()].unflatten(-1, (-1, 32)) * _power(scale.long() - 127)[..., None]
    return torch.where((scale == 255)[..., None], torch.full_like(v, float("nan")), v).flatten(-2)


def unpack_pages(k4, ks, v4, vs):
    """(k, v) float64 [pages, heads, 64, D] of one layer's pages, byte by byte from the layout's definition."""
    pages, heads, _, half = k4.shape
    d = 2 * half
    dev = k4.device
    k = torch.zeros(pages, heads, 64, d, dtype=torch.long, device=dev)
    v, s = torch.zeros_like(k), torch.zeros(pages, heads, 64, d // 32, dtype=torch.long, device=dev)
    for p in range(4):
        for j in range(d // 32):
            for i in range(8):
                byte = k4[..., p * (d // 8) + j * 4 + i // 2].long()
                k[..., 32 * j + 8 * p + i] = byte >> 4 * (i % 2) & 15
    for h in range(2):
        for p in range(4):
            for e in range(8):
                t = 32 * h + 16 * (e // 4) + 4 * p + e % 4
                for g in range(d // 32):
                    s[:, :, t, g] = vs[..., ((h * 4 + p) * (d // 32) + g) * 8 + e].long()
                    for n in range(16):
                        byte = v4[..., ((((h * (d // 64) + g // 2) * 4 + p) * 16 + n) * 2 + g % 2) * 8 + e].long()
                        v[:, :, t, 32 * g + n], v[:, :, t, 32 * g + 16 + n] = byte & 15, byte >> 4
    return values(k, ks.long()), values(v, s)


def slots(starts, lens, table, rows, pages):
    """For each row of a call its (page, place) or None; host lists."""
    out = [None] * rows
    for s in range(len(lens)):
        for r in range(starts[s], starts[s + 1]):
            pos = lens[s] - (starts[s + 1] - r)
            if 0 <= pos < 64 * len(table[s]) and 0 <= table[s][pos // 64] < pages:
                out[r] = (table[s][pos // 64], pos % 64)
    return out


def cache_attend(q, k, v, starts, lens, table, scale=None):
    """attend() of a call's rows over pages k, v [pages, heads, 64, D] of values: a row sees the tokens up to its own, of those
    that the table holds (its own may lie past it)."""
    heads, group = k.shape[1], q.shape[1] // k.shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    like = {}
    for s, n in enumerate(lens):
        count = starts[s + 1] - starts[s]
        if not count:
            continue
        first = n - count   # the first row's place
        n = min(max(n, 0), 64 * len(table[s]))
        at = [(table[s][t // 64], t % 64) for t in range(n)]
        held = torch.tensor([0 <= p < k.shape[0] for p, _ in at], dtype=torch.bool, device=q.device)
        page = torch.tensor([p if 0 <= p < k.shape[0] else 0 for p, _ in at], dtype=torch.long, device=q.device)
        place = torch.tensor([t for _, t in at], dtype=torch.long, device=q.device)
        see = (torch.arange(n, device=q.device) <= first + torch.arange(count, device=q.device)[:, None]) & held
        for h in range(q.shape[1]):
            r = attend(q[starts[s]:starts[s + 1], h], k[page, h // group, place], v[page, h // group, place], see, scale)
            for name, x in r.items():
                like.setdefault(name, torch.zeros(*q.shape[:2], x.shape[-1], dtype=torch.float64, device=q.device))
                like[name][starts[s]:starts[s + 1], h] = x
    del heads
    return like
