"""The block operators around the attention, as cases to time and compare: the residual stream's gated norm, rotary
positions, and linears with 4-bit weights.

- `norm`: s = residual_scale * x + branch_scale * gate * post(y), h = norm(s) * weight + bias, then
  h * (1 + scale) + shift: what stands between two sub-layers of a block (the branch's gate and norm, the residual
  addition, the next sub-layer's norm and its modulation), forward or with all gradients.
- `rotary`: the rotation of q and k by the positions of their tokens, in interleaved or half layout, on part of the head
  or all of it, on one axis or several, with stretched frequencies; forward or with gradients.
- `w4`: x w^T + bias where w is held as 4-bit codes with a scale (and, for integer codes, maybe a zero) for each group
  along K, from one row of x to a chunk's.

Sizes follow the 1.3B DiT that the other benchmarks use (1536 channels, 12 heads of 128, 8960 feed-forward channels,
chunks of 4 frames of 29 x 52 tokens, 512 context tokens) and generic ones around them.

With `own` false a pass computes the plain forms by elementary torch operations in 32 bits (angles in 64); with `own`
true it makes the framework's calls on the same inputs.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # e2m1 magnitudes of codes 0 .. 7; 8 .. 15 are their negatives
NIBBLES = {"int4": (0, 2, 4, 6, 1, 3, 5, 7), "fp4": (0, 1, 2, 3, 4, 5, 6, 7)}   # order of a word's 8 codes along K


def listed():
    return [
        # Between self-attention and the next sub-layer of a DiT block, a whole chunk: gated residual, LayerNorm,
        # shift and scale of each of the 4 frames. Bandwidth.
        {"name": "norm_chunk", "op": "norm", "batch": 1, "len": 6032, "width": 1536, "dtype": "bf16", "vec": "fp32",
         "norm": "layer", "post": "none", "mod": "frames", "groups": 4, "affine": False, "train": False},
        # The same in a training step: forward and the gradients of stream, branch, gate, shift and scale.
        {"name": "norm_chunk_train", "op": "norm", "batch": 1, "len": 6032, "width": 1536, "dtype": "bf16",
         "vec": "fp32", "norm": "layer", "post": "none", "mod": "frames", "groups": 4, "affine": False, "train": True},
        # One token of a decoder with RMS norms before and after its sub-layers. Latency.
        {"name": "norm_token", "op": "norm", "batch": 1, "len": 1, "width": 1536, "dtype": "bf16", "vec": "bf16",
         "norm": "rms", "post": "rms", "mod": "none", "groups": 1, "affine": True, "train": False},
        # Norms on both sides of the branch with learnt weights and a gate per channel, two ragged sequences, trained.
        {"name": "norm_sandwich_train", "op": "norm", "batch": 2, "len": 777, "width": 4096, "dtype": "fp16",
         "vec": "fp16", "norm": "rms", "post": "rms", "mod": "shared", "groups": 1, "affine": True, "train": True},
        # q and k of a chunk at its frame, row and column, deep into a rollout.
        {"name": "rotary_chunk", "op": "rotary", "batch": 1, "len": 6032, "q_heads": 12, "k_heads": 12, "dim": 128,
         "rot": 128, "axes": 3, "pairs": "interleaved", "dtype": "bf16", "reach": 1000, "stretch": 1.0,
         "train": False},
        # Grouped heads, half of each rotated, frequencies stretched for a long context; forward and gradients.
        {"name": "rotary_partial_train", "op": "rotary", "batch": 2, "len": 1999, "q_heads": 32, "k_heads": 8,
         "dim": 128, "rot": 64, "axes": 1, "pairs": "half", "dtype": "fp16", "reach": 131072, "stretch": 8.0,
         "train": True},
        # One new token for each of 64 sequences, far into their contexts. Latency.
        {"name": "rotary_tokens", "op": "rotary", "batch": 64, "len": 1, "q_heads": 12, "k_heads": 2, "dim": 128,
         "rot": 128, "axes": 1, "pairs": "half", "dtype": "bf16", "reach": 1000000, "stretch": 4.0, "train": False},
        # The time embedding's projection to a block's six modulation vectors: one row, all weights read.
        {"name": "w4_row", "op": "w4", "rows": 1, "in": 1536, "out": 9216, "fmt": "int4", "zero": False, "group": 128,
         "dtype": "bf16", "bias": True},
        # A few rows (sequences in decode) through the feed-forward's down projection, fp4 codes, small groups.
        {"name": "w4_few_fp4", "op": "w4", "rows": 5, "in": 8960, "out": 1536, "fmt": "fp4", "zero": False,
         "group": 32, "dtype": "bf16", "bias": False},
        # A batch of rows through the up projection, integer codes with zeros.
        {"name": "w4_batch", "op": "w4", "rows": 61, "in": 1536, "out": 8960, "fmt": "int4", "zero": True,
         "group": 64, "dtype": "fp16", "bias": True},
        # The text context's tokens through the cross-attention's key projection.
        {"name": "w4_context", "op": "w4", "rows": 512, "in": 1536, "out": 1536, "fmt": "int4", "zero": False,
         "group": 128, "dtype": "bf16", "bias": True},
        # A frame's tokens through the up projection: bound by the matrix cores.
        {"name": "w4_frame", "op": "w4", "rows": 1508, "in": 1536, "out": 8960, "fmt": "int4", "zero": True,
         "group": 128, "dtype": "bf16", "bias": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "rotary", "rotary", "w4", "w4"])
    if op == "norm":
        width = rng.choice([256, 384, 1000, 1024, 1536, 1536, 2048, 2056, 4096, 5120, 771])
        batch = rng.choice([1, 1, 2, 3])
        length = _log_int(rng, 1, max(2, 6032 * 1536 // (batch * width)))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        mod = rng.choice(["none", "shared", "frames", "frames"])
        return {"op": op, "batch": batch, "len": length, "width": width, "dtype": dtype,
                "vec": rng.choice([dtype, "fp32"]), "norm": rng.choice(["layer", "rms"]),
                "post": rng.choice(["none", "none", "layer", "rms"]), "mod": mod,
                "groups": rng.randint(1, min(5, length)) if mod == "frames" else 1,
                "affine": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "rotary":
        dim = rng.choice([64, 96, 128, 128, 256])
        k_heads = rng.choice([1, 2, 4, 8, 12])
        q_heads = k_heads * rng.choice([1, 2, 4])
        batch = rng.choice([1, 1, 2, 5, 32])
        length = _log_int(rng, 1, max(2, 6032 * 24 * 128 // (2 * batch * (q_heads + k_heads) * dim)))
        axes = rng.choice([1, 1, 3])
        return {"op": op, "batch": batch, "len": length, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
                "rot": dim if axes == 3 else rng.choice([dim, dim, dim // 2, 24]), "axes": axes,
                "pairs": rng.choice(["interleaved", "half"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "reach": _log_int(rng, 100, 1000000), "stretch": rng.choice([1.0, 1.0, 2.5, 8.0]),
                "train": rng.random() < 0.4}
    k, n = rng.choice([(1536, 1536), (1536, 8960), (8960, 1536), (1536, 9216), (2048, 1024), (1000, 1003), (256, 64)])
    fmt = rng.choice(["int4", "int4", "fp4"])
    return {"op": op, "rows": _log_int(rng, 1, 1508), "in": k, "out": n, "fmt": fmt,
            "zero": fmt == "int4" and rng.random() < 0.5, "group": rng.choice([32, 64, 128]),
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "bias": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs


class _Rand:
    def __init__(self, seed):
        self.device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.gen = torch.Generator(device=self.device).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.gen, device=self.device) * std + mean).to(dtype)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device=self.device)


def _group_len(case):
    return -(-case["len"] // case["groups"])


def _prepare_norm(case, seed):
    r = _Rand(seed)
    b, n, c = case["batch"], case["len"], case["width"]
    t, v = DTYPES[case["dtype"]], DTYPES[case["vec"]]
    # channels of a residual stream differ in size, and a few are far larger than the rest
    size = torch.exp(r.normal(c, std=0.5))
    a = {"x": (r.normal(b, n, c, std=1.5, mean=0.1) * size).to(t), "y": r.normal(b, n, c, dtype=t)}
    mods = {"none": None, "shared": (c,), "frames": (b, case["groups"], c)}[case["mod"]]
    if mods is not None:
        # as the program has them: three of the six vectors that one projection gives for each frame
        six = r.normal(*mods[:-1], 6, c, std=0.3, dtype=v)
        a["gate"], a["shift"], a["scale"] = six[..., 2, :], six[..., 3, :], six[..., 4, :]
    if case["affine"]:
        a["weight"] = r.normal(c, std=0.2, mean=1.0, dtype=v)
        if case["norm"] == "layer":
            a["bias"] = r.normal(c, std=0.2, dtype=v)
        if case["post"] != "none":
            a["post_weight"] = r.normal(c, std=0.2, mean=1.0, dtype=v)
    state = {"case": case, "args": a, "residual_scale": 1.0, "branch_scale": 1.0 if mods is not None else 0.7}
    if case["train"]:
        state["args"] = {k: x.detach().requires_grad_() for k, x in a.items()}
        state["grads"] = (r.normal(b, n, c, std=0.05, dtype=t), r.normal(b, n, c, std=0.05, dtype=t))
    return state


def _sections(case):
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return (pairs,)
    side = pairs // 3
    return (pairs - 2 * side, side, side)


def _prepare_rotary(case, seed):
    r = _Rand(seed)
    b, n, d, t = case["batch"], case["len"], case["dim"], DTYPES[case["dtype"]]
    q = r.normal(b, n, case["q_heads"], d, dtype=t)
    k = r.normal(b, n, case["k_heads"], d, dtype=t)
    start = r.ints(0, case["reach"], b, 1)
    count = torch.arange(n, device=r.device)
    if case["axes"] == 1:
        pos = start + count
    else:   # frame, row and column of each token of a grid as wide as the DiT's
        pos = torch.stack((start + count // 1508, (count // 52 % 29).expand(b, n), (count % 52).expand(b, n)), dim=-1)
    # each axis has frequencies of its own; past the trained length the slow ones are stretched and the fast ones kept,
    # with a ramp between (64 bits: far positions lose the angle otherwise)
    freq, axis = [], []
    for i, pairs in enumerate(_sections(case)):
        f = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=r.device) / pairs)
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freq.append(f * keep + f / case["stretch"] * (1 - keep))
        axis += [i] * pairs
    state = {"case": case, "q": q, "k": k, "pos": pos, "freq": torch.cat(freq),
             "axis": torch.tensor(axis, dtype=torch.int32, device=r.device) if case["axes"] > 1 else None,
             "factor": 1.0 + 0.1 * math.log(case["stretch"])}
    if case["train"]:
        q.requires_grad_()
        k.requires_grad_()
        state["grads"] = (r.normal(*q.shape, std=0.05, dtype=t), r.normal(*k.shape, std=0.05, dtype=t))
    return state


def _prepare_w4(case, seed):
    r = _Rand(seed)
    k, n, g, t = case["in"], case["out"], case["group"], DTYPES[case["dtype"]]
    kp, np_ = -(-k // 128) * 128, -(-n // 16) * 16
    w = torch.zeros(np_, kp, device=r.device)
    w[:n, :k] = r.normal(n, k, std=k ** -0.5)
    w = w.view(np_, kp // g, g)
    # codes and scales as a checkpoint holds them
    zero = None
    if case["fmt"] == "fp4":
        scale = (w.abs().amax(2, keepdim=True) / 6).to(torch.bfloat16)
        mids = torch.tensor([(a + b) / 2 for a, b in zip(FP4, FP4[1:])], device=r.device)
        u = torch.where(scale > 0, w / scale.float(), torch.zeros_like(w))
        codes = torch.bucketize(u.abs(), mids) + 8 * (u < 0)
    elif case["zero"]:
        lo, hi = w.amin(2, keepdim=True).clamp(max=0), w.amax(2, keepdim=True).clamp(min=0)
        scale = ((hi - lo) / 15).to(torch.bfloat16)
        u = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(lo))
        zero = (-lo * u).round().clamp(0, 15)
        codes = (w * u + zero).round().clamp(0, 15)
    else:
        scale = (w.abs().amax(2, keepdim=True) / 7).to(torch.bfloat16)
        u = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(scale.float()))
        codes = (w * u + 8).round().clamp(0, 15)
    codes = codes.to(torch.uint8).view(np_, kp)
    # the same laid out once for the kernel: tiles of 16 rows x 128 columns, word j of lane (row, quarter) the 8 codes
    # from column 32 j + 8 quarter on
    tiles = codes.view(np_ // 16, 16, kp // 128, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)[..., NIBBLES[case["fmt"]]]
    packed = (tiles[..., 0::2] | tiles[..., 1::2] << 4).reshape(np_ // 16, kp // 128, 1024).contiguous()

    def per_tile(s):
        return s.view(np_ // 16, 16, kp // 128, 128 // g).transpose(1, 2).contiguous()

    zero = zero.to(torch.uint8) if zero is not None else None
    return {"case": case, "x": r.normal(case["rows"], k, dtype=t), "bias": r.normal(n, std=0.1, dtype=t)
            if case["bias"] else None, "codes": codes[:n], "scale": scale[:n, :, 0],
            "zero": zero[:n, :, 0] if zero is not None else None, "packed": packed, "tile_scale": per_tile(scale),
            "tile_zero": per_tile(zero) if zero is not None else None}


def prepare(case, seed):
    return {"norm": _prepare_norm, "rotary": _prepare_rotary, "w4": _prepare_w4}[case["op"]](case, seed)


# ---------------------------------------------------------------- one pass


def _normed(x, kind, eps=1e-6):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def _tokens(v, case):
    """A modulation vector for each token: [C], or [B, groups, C] repeated over the group's tokens."""
    v = v.float()
    return v if v.dim() == 1 else v.repeat_interleave(_group_len(case), dim=1)[:, :case["len"]]


def _plain_norm(state):
    case, a = state["case"], state["args"]
    p = _normed(a["y"].float(), case["post"])
    if "post_weight" in a:
        p = p * a["post_weight"].float()
    if "gate" in a:
        p = p * _tokens(a["gate"], case)
    s = state["residual_scale"] * a["x"].float() + state["branch_scale"] * p
    h = _normed(s, case["norm"])
    if "weight" in a:
        h = h * a["weight"].float()
    if "bias" in a:
        h = h + a["bias"].float()
    if "scale" in a:
        h = h * (1 + _tokens(a["scale"], case)) + _tokens(a["shift"], case)
    return s.to(a["x"].dtype), h.to(a["x"].dtype)


def _own_norm(state):
    from lingbot_world_v2_realtime_amd.layers.norm import gated_norm
    case = state["case"]
    return gated_norm(**state["args"], norm=case["norm"], post_norm=None if case["post"] == "none" else case["post"],
                      residual_scale=state["residual_scale"], branch_scale=state["branch_scale"],
                      group_len=_group_len(case) if case["mod"] == "frames" else None)


def _plain_rotary(state):
    case = state["case"]
    rot, pos = case["rot"], state["pos"].double()
    pos = pos[..., None] if state["axis"] is None else pos[..., state["axis"].long()]
    ang = pos * state["freq"]
    cos, sin = (f(ang).mul(state["factor"]).float()[:, :, None] for f in (torch.cos, torch.sin))

    def turn(x):
        y, rest = x[..., :rot].float(), x[..., rot:]
        if case["pairs"] == "interleaved":
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((y.to(x.dtype), rest), dim=-1)

    return turn(state["q"]), turn(state["k"])


def _own_rotary(state):
    from lingbot_world_v2_realtime_amd.layers.rotary import Rotary, rotary_embed
    rope = Rotary(state["freq"], state["axis"], state["case"]["pairs"], state["factor"])
    return rotary_embed(state["q"], state["k"], state["pos"], rope)


def _plain_w4(state):
    case, g = state["case"], state["case"]["group"]
    codes = state["codes"]
    if case["fmt"] == "fp4":
        w = torch.tensor(FP4 + tuple(-x for x in FP4), device=codes.device)[codes.int()]
    else:
        w = codes.float() - (8.0 if state["zero"] is None else state["zero"].float().repeat_interleave(g, dim=1))
    w = (w * state["scale"].float().repeat_interleave(g, dim=1))[:, :case["in"]]
    y = state["x"].float() @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _own_w4(state):
    from lingbot_world_v2_realtime_amd import kernels
    case = state["case"]
    return kernels.gemm_w4(state["x"], state["packed"], state["tile_scale"], state["tile_zero"], state["bias"],
                           out_features=case["out"], fmt=case["fmt"])


def run(state):
    case = state["case"]
    if case["op"] == "w4":
        return _own_w4(state) if own else _plain_w4(state)
    if case["op"] == "norm":
        out = _own_norm(state) if own else _plain_norm(state)
        leaves = state["args"]
    else:
        out = _own_rotary(state) if own else _plain_rotary(state)
        leaves = {"q": state["q"], "k": state["k"]}
    if not case["train"]:
        return list(out)
    grads = torch.autograd.grad(out, list(leaves.values()), state["grads"])
    return {"out": [o.detach() for o in out], **{"d_" + k: g for k, g in zip(leaves, grads)}}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "norm":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        cells = case["batch"] * case["len"] * case["width"]
        vecs = {"none": 0, "shared": 3, "frames": 3 * case["batch"] * case["groups"]}[case["mod"]] + 3 * case["affine"]
        small = vecs * case["width"] * DTYPES[case["vec"]].itemsize
        # x, y -> s, h; trained: also ds, dh -> dx, dy (x and y are read once in a pass that did both)
        return {"bytes": cells * size * (8 if case["train"] else 4) + small * (2 if case["train"] else 1),
                "flops": cells * (50 if case["train"] else 15)}
    if case["op"] == "rotary":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        cells = case["batch"] * case["len"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        times = 2 if case["train"] else 1
        return {"bytes": times * 2 * cells * size + 8 * case["batch"] * case["len"] * case["axes"],
                "flops": times * 3 * cells * case["rot"] // case["dim"]}
    m, k, n = case["rows"], case["in"], case["out"]
    weights = n * k // 2 + n * -(-k // case["group"]) * (3 if case["zero"] else 2)
    return {"bytes": weights + 2 * (m * k + m * n + n * case["bias"]), "flops": 2 * m * k * n}


# ---------------------------------------------------------------- the definitions in 64 bits


def _stats64(x, kind, eps=1e-6):
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else torch.zeros_like(x[..., :1])
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    return mean, 1 / torch.sqrt(var + eps)


def _norm_grad64(d, unit, r, kind):
    """Gradient through unit = (x - mean) r, given that of unit."""
    d = d - unit * (d * unit).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - d.mean(-1, keepdim=True)
    return d * r


def _exact_norm(state):
    case = state["case"]
    b, n, c = case["batch"], case["len"], case["width"]
    a = {k: v.detach().double() for k, v in state["args"].items()}
    row = torch.arange(n, device=a["x"].device) // _group_len(case)

    def at(name, other):
        v = a.get(name)
        return other if v is None else v if v.dim() == 1 else v[:, row]

    def back(name, d):
        """The gradient of vector `name` from that of its every use."""
        v = state["args"][name]
        if v.dim() == 1:
            out = d.sum((0, 1))
        else:
            out = torch.zeros_like(v, dtype=torch.float64)
            out.index_add_(1, row, d)
        return out

    al, be = state["residual_scale"], state["branch_scale"]
    y, one = a["y"], torch.ones(c, dtype=torch.float64, device=row.device)
    if case["post"] == "none":
        yu, yr = y, None
    else:
        ym, yr = _stats64(y, case["post"])
        yu = (y - ym) * yr
    pw, gate = at("post_weight", one), at("gate", one)
    s = al * a["x"] + be * gate * pw * yu
    sm, sr = _stats64(s, case["norm"])
    su = (s - sm) * sr
    w, mul = at("weight", one), 1 + at("scale", 0 * one)
    lin = su * w + at("bias", 0 * one)
    h = lin * mul + at("shift", 0 * one)
    if not case["train"]:
        return [s, h]
    ds, dh = (g.double() for g in state["grads"])
    ds = ds + _norm_grad64(dh * mul * w, su, sr, case["norm"])
    dyu = ds * be * gate * pw
    each = {"x": al * ds, "y": dyu if yr is None else _norm_grad64(dyu, yu, yr, case["post"]),
            "gate": ds * be * pw * yu, "post_weight": ds * be * gate * yu, "weight": dh * mul * su, "bias": dh * mul,
            "scale": dh * lin, "shift": dh}
    return {"out": [s, h], **{"d_" + k: each[k] if k in ("x", "y") else back(k, each[k]) for k in a}}


def _exact_rotary(state):
    case = state["case"]
    half, pos = case["rot"] // 2, state["pos"]
    which = torch.zeros(half, dtype=torch.long, device=pos.device) if state["axis"] is None else state["axis"].long()
    pos = pos[..., None] if state["axis"] is None else pos
    turn = torch.polar(torch.full((), state["factor"], dtype=torch.float64, device=pos.device),
                       pos[..., which].double() * state["freq"])[:, :, None]
    first = torch.arange(half, device=pos.device)
    first, second = (2 * first, 2 * first + 1) if case["pairs"] == "interleaved" else (first, first + half)

    def apply(x, by):
        x = x.detach().double()
        out = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * by
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out = [apply(state["q"], turn), apply(state["k"], turn)]
    if not case["train"]:
        return out
    dq, dk = (apply(g, turn.conj()) for g in state["grads"])
    return {"out": out, "d_q": dq, "d_k": dk}


def _exact_w4(state):
    case = state["case"]
    n, k, g = case["out"], case["in"], case["group"]
    codes, scale = state["codes"].long(), state["scale"].double()
    if case["fmt"] == "fp4":   # sign, two exponent bits, one mantissa bit
        sign, e, m = codes >> 3, codes >> 1 & 3, codes & 1
        mag = torch.where(e > 0, (2 + m).double() * 2.0 ** (e - 2).double(), 0.5 * m.double())
        value = torch.where(sign > 0, -mag, mag)
    else:
        off = torch.full_like(scale, 8) if state["zero"] is None else state["zero"].double()
        value = (codes.view(n, -1, g).double() - off[:, :, None]).view(n, -1)
    w = value.view(n, -1, g) * scale[:, :, None]
    y = torch.matmul(state["x"].double(), w.reshape(n, -1)[:, :k].t().contiguous())
    return y if state["bias"] is None else y + state["bias"].double()


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "rotary": _exact_rotary, "w4": _exact_w4}[case["op"]](state)
