"""Causal self-attention from its projections to a cache held in 4 bits, as cases to time and compare.

- `norm_rotary`: the RMS norm of every head of q and k with learnt weights, and the rotation by the tokens' positions;
  forward or with all gradients.
- `attention`: causal attention over sequences of different lengths packed one behind the other, a head of k and v for one
  or several heads of q, keys from before the first query or fewer than the queries; forward or with gradients.
- `cache_write`: the K and V of each sequence's newest tokens into pages of 64 tokens of a cache that holds e2m1 codes
  with a power-of-two scale for each 32 channels of a token, and what the cache then holds of them.
- `cache_attend`: attention of each sequence's newest tokens (one, or a few) over all that its pages hold.

Sizes follow the 1.3B DiT that the other benchmarks use (12 heads of 128, chunks of 6032 tokens in 4 frames of 29 x 52,
24128 tokens attended, 512 context tokens, captions of 77) and generic ones with grouped heads around them.

With `own` false a pass computes the plain forms by elementary torch operations in 32 bits (angles in 64); with `own`
true it makes the framework's calls on the same inputs.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # e2m1 magnitudes of codes 0 .. 7; 8 .. 15 are their negatives
PAGE = 64                                        # tokens of a page
EPS = 1e-6


def listed():
    return [
        # q and k of a DiT block's chunk, normed by head and turned by frame, row and column. Bandwidth.
        {"name": "norm_rotary_chunk", "op": "norm_rotary", "batch": 1, "len": 6032, "q_heads": 12, "k_heads": 12,
         "dim": 128, "rot": 128, "axes": 3, "pairs": "interleaved", "dtype": "bf16", "weight": "bf16", "reach": 1000,
         "train": False},
        # Grouped heads in a training step, two ragged rows of tokens, fp32 weights: forward and every gradient.
        {"name": "norm_rotary_train", "op": "norm_rotary", "batch": 2, "len": 1999, "q_heads": 32, "k_heads": 8,
         "dim": 128, "rot": 64, "axes": 1, "pairs": "half", "dtype": "bf16", "weight": "fp32", "reach": 131072,
         "train": True},
        # One new token for each of 64 sequences. Latency.
        {"name": "norm_rotary_tokens", "op": "norm_rotary", "batch": 64, "len": 1, "q_heads": 12, "k_heads": 2,
         "dim": 128, "rot": 128, "axes": 1, "pairs": "half", "dtype": "bf16", "weight": "bf16", "reach": 1000000,
         "train": False},
        # A batch of prompts of very different lengths, grouped heads.
        {"name": "attention_prompts", "op": "attention", "seqs": 8, "longest": 1508, "q_heads": 32, "k_heads": 8,
         "dim": 128, "prefix": 0, "tail": 5, "dtype": "bf16", "train": False},
        # One long sequence, two chunks of a rollout: the matrix cores.
        {"name": "attention_long", "op": "attention", "seqs": 1, "longest": 12064, "q_heads": 12, "k_heads": 12,
         "dim": 128, "prefix": 0, "tail": 0, "dtype": "bf16", "train": False},
        # Many captions, heads of 64 channels: few rows each, mostly masked tiles.
        {"name": "attention_captions", "op": "attention", "seqs": 61, "longest": 77, "q_heads": 16, "k_heads": 16,
         "dim": 64, "prefix": 0, "tail": 0, "dtype": "fp16", "train": False},
        # A training step over packed documents, grouped heads: forward and gradients.
        {"name": "attention_train", "op": "attention", "seqs": 5, "longest": 1508, "q_heads": 12, "k_heads": 4,
         "dim": 128, "prefix": 0, "tail": 3, "dtype": "bf16", "train": True},
        # Prompts into the cache.
        {"name": "cache_write_prompts", "op": "cache_write", "seqs": 4, "longest": 3016, "held": 100, "k_heads": 8,
         "dim": 128, "dtype": "bf16"},
        # One new token of each of 64 sequences into the cache. Latency.
        {"name": "cache_write_tokens", "op": "cache_write", "seqs": 64, "longest": 1, "held": 777, "k_heads": 8,
         "dim": 128, "dtype": "bf16"},
        # A single sequence's next token over a frame of tokens. Latency.
        {"name": "cache_attend_token", "op": "cache_attend", "seqs": 1, "longest": 1508, "tokens": 1, "q_heads": 12,
         "k_heads": 4, "dim": 128, "dtype": "bf16"},
        # The next token of 61 sequences of very different lengths.
        {"name": "cache_attend_batch", "op": "cache_attend", "seqs": 61, "longest": 6032, "tokens": 1, "q_heads": 32,
         "k_heads": 8, "dim": 128, "dtype": "bf16"},
        # Five drafted tokens of each of 7 long sequences, checked at once.
        {"name": "cache_attend_drafts", "op": "cache_attend", "seqs": 7, "longest": 24128, "tokens": 5, "q_heads": 12,
         "k_heads": 12, "dim": 128, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rotary", "attention", "attention", "cache_write", "cache_attend", "cache_attend"])
    k_heads = rng.choice([1, 2, 4, 8, 12])
    q_heads = k_heads * rng.choice([1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm_rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        batch = rng.choice([1, 1, 2, 5, 32])
        axes = rng.choice([1, 1, 3])
        length = _log_int(rng, 1, max(2, 6032 * 24 * 128 // (2 * batch * (q_heads + k_heads) * dim)))
        dtype = rng.choice([dtype, dtype, "fp32"])
        return {"op": op, "batch": batch, "len": length, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
                "rot": dim if axes == 3 else rng.choice([dim, dim, dim // 2, 24]), "axes": axes,
                "pairs": rng.choice(["interleaved", "half"]), "dtype": dtype, "weight": rng.choice([dtype, "fp32"]),
                "reach": _log_int(rng, 100, 1000000), "train": rng.random() < 0.4}
    dim = rng.choice([64, 128, 128])
    if op == "attention":
        seqs = _log_int(rng, 1, 61)
        # the padded plain form's products stay below the longest listed one's
        most = int(math.sqrt(12064 ** 2 * 12 * 128 / (4 * seqs * q_heads * dim)))
        return {"op": op, "seqs": seqs, "longest": _log_int(rng, 1, min(most, 6032)), "q_heads": q_heads,
                "k_heads": k_heads, "dim": dim, "prefix": rng.choice([0, 0, 0, 33, 512, -7]),
                "tail": rng.choice([0, 0, 1, 70]), "dtype": dtype, "train": rng.random() < 0.4}
    if op == "cache_write":
        seqs = _log_int(rng, 1, 64)
        return {"op": op, "seqs": seqs, "longest": _log_int(rng, 1, max(2, 6032 * 2 // seqs)),
                "held": _log_int(rng, 1, 1508) - 1, "k_heads": k_heads, "dim": dim, "dtype": dtype}
    seqs = _log_int(rng, 1, 64)
    tokens = rng.choice([1, 1, 1, 2, 5, 16])
    return {"op": op, "seqs": seqs, "longest": _log_int(rng, tokens, max(tokens + 1, min(24128, 6032 * 61 * 4 // (seqs * k_heads)))),
            "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "dtype": dtype}


# ---------------------------------------------------------------- inputs


class _Rand:
    def __init__(self, seed):
        self.device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.gen = torch.Generator(device=self.device).manual_seed(int(seed))

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.gen, device=self.device) * std + mean).to(dtype)

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.gen, device=self.device)


def _lengths(case, least):
    """Lengths between `least` and the longest, spread evenly in an order of their own; the first is the longest."""
    return [case["longest"] - int((case["longest"] - least) * (i * 0.6180339887498949 % 1.0)) for i in range(case["seqs"])]


def _starts(lens, device):
    return torch.tensor([0] + lens, device=device).cumsum(0).to(torch.int32)


def _sections(case):
    pairs = case["rot"] // 2
    if case["axes"] == 1:
        return (pairs,)
    side = pairs // 3
    return (pairs - 2 * side, side, side)


def _prepare_norm_rotary(case, seed):
    r = _Rand(seed)
    b, n, d, t, w = case["batch"], case["len"], case["dim"], DTYPES[case["dtype"]], DTYPES[case["weight"]]
    # a projection's channels differ in size; q and k are parts of one projection
    size = torch.exp(r.normal(case["q_heads"] + case["k_heads"], d, std=0.5))
    both = (r.normal(b, n, case["q_heads"] + case["k_heads"], d) * size).to(t)
    q, k = both[:, :, :case["q_heads"]], both[:, :, case["q_heads"]:]
    start = r.ints(0, case["reach"], b, 1)
    count = torch.arange(n, device=r.device)
    if case["axes"] == 1:
        pos = start + count
    else:   # frame, row and column of each token of a grid as wide as the DiT's
        pos = torch.stack((start + count // 1508, (count // 52 % 29).expand(b, n), (count % 52).expand(b, n)), dim=-1)
    freq, axis = [], []
    for i, pairs in enumerate(_sections(case)):
        freq.append(10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=r.device) / pairs))
        axis += [i] * pairs
    state = {"case": case, "q": q, "k": k, "pos": pos, "freq": torch.cat(freq),
             "axis": torch.tensor(axis, dtype=torch.int32, device=r.device) if case["axes"] > 1 else None,
             "q_weight": r.normal(d, std=0.3, mean=1.0, dtype=w), "k_weight": r.normal(d, std=0.3, mean=1.0, dtype=w)}
    if case["train"]:
        for name in ("q", "k", "q_weight", "k_weight"):
            state[name] = state[name].detach().requires_grad_()
        state["grads"] = (r.normal(*q.shape, std=0.05, dtype=t), r.normal(*k.shape, std=0.05, dtype=t))
    return state


def _attention_lens(case):
    """Queries and keys of each sequence."""
    lens = _lengths(case, min(1, case["longest"]))
    return lens, [max(0, n + case["prefix"]) for n in lens]


def _prepare_attention(case, seed):
    r = _Rand(seed)
    lens, k_lens = _attention_lens(case)
    t, d = DTYPES[case["dtype"]], case["dim"]
    rows, k_rows = sum(lens) + case["tail"], sum(k_lens) + case["tail"]
    state = {"case": case, "q": r.normal(rows, case["q_heads"], d, std=1.2, dtype=t),
             "k": (r.normal(k_rows, case["k_heads"], d) + r.normal(case["k_heads"], d, std=0.5)).to(t),
             "v": r.normal(k_rows, case["k_heads"], d, dtype=t), "starts": _starts(lens, r.device),
             "k_starts": _starts(k_lens, r.device)}
    if case["train"]:
        for name in ("q", "k", "v"):
            state[name].requires_grad_()
        state["grad"] = r.normal(rows, case["q_heads"], d, std=0.05, dtype=t)
    return state


def _encode(x):
    """e2m1 codes (uint8) and E8M0 scales (uint8, of each 32 channels) of x [..., D], in bf16 or fp16: the least power of two
    that leaves no magnitude over 6, codes to the nearest value, ties to the even code."""
    g = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = (e - torch.where(m <= 0.75, 3, 2)).clamp(min=-125)
    u = torch.ldexp(g, -e)
    mag = u.abs()
    code = ((mag > 0.25).byte() + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75) + (mag > 2.5) + (mag >= 3.5) + (mag > 5.0)
            + 8 * torch.signbit(u).byte())
    return code.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _pages(case, lens, r):
    """A table of shuffled pages for sequences of `lens` tokens, with a few pages that nobody holds, and how many there are."""
    counts = [-(-n // PAGE) for n in lens]
    total = sum(counts) + 3
    order = torch.randperm(total, generator=r.gen, device=r.device).to(torch.int32)
    table = torch.zeros(len(lens), max(max(counts), 1), dtype=torch.int32, device=r.device)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _k_page(codes, scale):
    """Codes [pages, heads, 64, D] and scales [pages, heads, 64, D / 32] as the cache has them: a token's codes in four
    parts, part p holding channels 32 j + 8 p .. + 8 of every j; two codes a byte, the lower channel in the low bits."""
    c = codes.unflatten(-1, (-1, 4, 8)).transpose(-3, -2)
    return (c[..., 0::2] | c[..., 1::2] << 4).flatten(-3).contiguous(), scale.contiguous()


def _v_page(codes, scale):
    """The same for V: byte [half][D / 64][part p][channel n][group][e] holds the codes of token 32 half + 16 (e / 4) + 4 p +
    e % 4 at channels 32 g + n (low bits) and 32 g + 16 + n, g the group of the 64 channels; scales [half][p][D / 32][e]."""
    pages, heads, _, d = codes.shape
    c = codes.view(pages, heads, 2, 2, 4, 4, d // 64, 2, 2, 16)   # half, e / 4, p, e % 4, D / 64, group, low or high, n
    c = (c[..., 0, :] | c[..., 1, :] << 4).permute(0, 1, 2, 6, 4, 8, 7, 3, 5)
    s = scale.view(pages, heads, 2, 2, 4, 4, d // 32).permute(0, 1, 2, 4, 6, 3, 5)
    return c.reshape(pages, heads, 32 * d).contiguous(), s.reshape(pages, heads, 2 * d).contiguous()


def _prepare_cache_write(case, seed):
    r = _Rand(seed)
    new = _lengths(case, min(1, case["longest"]))
    lens = [n + (case["held"] * (i + 1)) // case["seqs"] for i, n in enumerate(new)]
    t, d, h = DTYPES[case["dtype"]], case["dim"], case["k_heads"]
    table, pages = _pages(case, lens, r)
    k = (r.normal(sum(new), h, d) + r.normal(h, d, std=1.5)).to(t)
    u8 = {"dtype": torch.uint8, "device": r.device}
    return {"case": case, "k": k, "v": r.normal(sum(new), h, d, dtype=t), "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device=r.device), "starts": _starts(new, r.device),
            # one layer of what the program's cache holds, in the kernels' layout ...
            "cache": (torch.zeros(1, pages, h, PAGE, d // 2, **u8), torch.zeros(1, pages, h, PAGE, d // 32, **u8),
                      torch.zeros(1, pages, h, PAGE * d // 2, **u8), torch.zeros(1, pages, h, PAGE * d // 32, **u8)),
            # ... and for the plain form, which holds a code a byte
            "codes": [torch.zeros(pages, h, PAGE, n, **u8) for n in (d, d // 32, d, d // 32)]}


def _prepare_cache_attend(case, seed):
    r = _Rand(seed)
    lens = _lengths(case, case["tokens"])
    t, d, h = DTYPES[case["dtype"]], case["dim"], case["k_heads"]
    table, pages = _pages(case, lens, r)
    k = _encode((r.normal(pages, h, PAGE, d) + r.normal(h, 1, d, std=1.5)).to(torch.bfloat16))
    v = _encode(r.normal(pages, h, PAGE, d).to(torch.bfloat16))
    cache = tuple(x[None] for x in (*_k_page(*k), *_v_page(*v)))
    return {"case": case, "q": r.normal(case["seqs"] * case["tokens"], case["q_heads"], d, std=1.2, dtype=t), "table": table,
            "lens": torch.tensor(lens, dtype=torch.int32, device=r.device),
            "starts": _starts([case["tokens"]] * case["seqs"], r.device), "cache": cache, "codes": [*k, *v]}


def prepare(case, seed):
    return {"norm_rotary": _prepare_norm_rotary, "attention": _prepare_attention, "cache_write": _prepare_cache_write,
            "cache_attend": _prepare_cache_attend}[case["op"]](case, seed)


# ---------------------------------------------------------------- one pass


def _plain_norm_rotary(state):
    case = state["case"]
    rot, pos = case["rot"], state["pos"].double()
    pos = pos[..., None] if state["axis"] is None else pos[..., state["axis"].long()]
    ang = pos * state["freq"]
    cos, sin = torch.cos(ang).float()[:, :, None], torch.sin(ang).float()[:, :, None]

    def turn(x, w):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.float()
        y, rest = y[..., :rot], y[..., rot:]
        if case["pairs"] == "interleaved":
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:]
            y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
        return torch.cat((y, rest), dim=-1).to(x.dtype)

    return turn(state["q"], state["q_weight"]), turn(state["k"], state["k_weight"])


def _own_norm_rotary(state):
    from lingbot_world_v2_realtime_amd.layers.rotary import Rotary, norm_rotary_embed
    rope = Rotary(state["freq"], state["axis"], state["case"]["pairs"])
    return norm_rotary_embed(state["q"], state["k"], state["pos"], rope, state["q_weight"], state["k_weight"], EPS)


def _padded(x, starts, longest):
    """Packed rows [T, H, D] as [S, H, longest, D] with zeros behind each sequence, and where each row of the padded form
    comes from."""
    at = starts[:-1, None].long() + torch.arange(longest, device=x.device)
    held = at < starts[1:, None]
    at = at.clamp(max=max(x.shape[0] - 1, 0))
    return torch.where(held[..., None, None], x[at], torch.zeros((), device=x.device)).transpose(1, 2), at, held


def _softmax_product(logits, see, v):
    """softmax over the keys that `see` leaves, times v; a row that sees none gives 0."""
    logits = logits.masked_fill(~see, -math.inf)
    top = logits.detach().amax(-1, keepdim=True) if logits.shape[-1] else logits.new_zeros(*logits.shape[:-1], 1)
    p = torch.exp(logits - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    return (p / total.masked_fill(total == 0, 1.0)) @ v


def _plain_attention(state):
    case = state["case"]
    q, starts, k_starts = state["q"].float(), state["starts"], state["k_starts"]
    longest, k_longest = case["longest"], max(0, case["longest"] + case["prefix"])
    if not k_longest:
        return (q * 0).to(state["q"].dtype)
    qp, at, held = _padded(q, starts, longest)
    (kp, _, k_held), (vp, _, _) = (_padded(state[n].float(), k_starts, k_longest) for n in ("k", "v"))
    qp = qp.unflatten(1, (case["k_heads"], -1))                                        # [S, Hk, G, L, D]
    logits = qp.flatten(2, 3) @ kp.transpose(2, 3).contiguous() * case["dim"] ** -0.5   # [S, Hk, G L, Lk]
    i, j = torch.arange(longest, device=q.device), torch.arange(k_longest, device=q.device)
    shift = (k_starts[1:] - k_starts[:-1]) - (starts[1:] - starts[:-1])                # the last query is at the last key
    see = (j <= i[:, None] + shift[:, None, None]) & k_held[:, None]                   # [S, L, Lk]
    out = _softmax_product(logits.unflatten(2, qp.shape[2:4]), see[:, None, None], vp[:, :, None])
    out = out.flatten(1, 2).transpose(1, 2)
    return torch.zeros_like(q).index_put((at[held],), out[held]).to(state["q"].dtype)


def _own_attention(state):
    from lingbot_world_v2_realtime_amd.layers.packed import packed_attention
    return packed_attention(state["q"], state["k"], state["v"], state["starts"], state["k_starts"])


def _values(codes, scale):
    """What codes [..., D] with scales [..., D / 32] stand for, in fp32."""
    table = torch.tensor(FP4 + tuple(-x for x in FP4), device=codes.device)
    return torch.ldexp(table[codes.int()].unflatten(-1, (-1, 32)), scale.int()[..., None] - 127).flatten(-2)


def _token_slots(state):
    """Page and place in it of every token of the call: each sequence's newest."""
    starts, lens = state["starts"].long(), state["lens"].long()
    t = torch.arange(state["k"].shape[0], device=starts.device)
    s = torch.searchsorted(starts, t, right=True) - 1
    pos = lens[s] - (starts[s + 1] - t)
    return state["table"][s, pos // PAGE].long(), pos % PAGE


def _plain_cache_write(state):
    page, place = _token_slots(state)
    out = []
    for x, codes, scale in ((state["k"], *state["codes"][:2]), (state["v"], *state["codes"][2:])):
        new = _encode(x)
        codes[page, :, place], scale[page, :, place] = new
        out.append(_values(codes[page, :, place], scale[page, :, place]).to(torch.bfloat16))
    return out


def _own_cache_write(state):
    from lingbot_world_v2_realtime_amd.layers.kv4 import KV4Cache
    cache = KV4Cache(*state["cache"])
    cache.write(0, state["k"], state["v"], state["table"], state["lens"], state["starts"])
    return list(cache.read(0, state["table"], state["lens"], state["starts"], tokens=state["k"].shape[0]))


def _plain_cache_attend(state):
    case, table = state["case"], state["table"].long()
    lens, n = state["lens"].long(), case["tokens"]

    def gathered(codes, scale):   # [S, Hk, pages of the longest * 64, D]
        x = _values(codes[table], scale[table])
        return x.transpose(1, 2).flatten(2, 3)

    k, v = gathered(*state["codes"][:2]), gathered(*state["codes"][2:])
    q = state["q"].float().view(case["seqs"], n, case["k_heads"], -1, case["dim"]).permute(0, 2, 3, 1, 4)
    logits = q.flatten(2, 3) @ k.transpose(2, 3).contiguous() * case["dim"] ** -0.5
    j, i = torch.arange(k.shape[2], device=k.device), torch.arange(n, device=k.device)
    see = j < lens[:, None, None] - (n - 1 - i[:, None])   # [S, n, Lk]
    see = see[:, None, None].expand(-1, 1, q.shape[2], -1, -1).flatten(2, 3)
    out = _softmax_product(logits, see, v).unflatten(2, (-1, n))
    return out.permute(0, 3, 1, 2, 4).reshape(state["q"].shape).to(state["q"].dtype)


def _own_cache_attend(state):
    from lingbot_world_v2_realtime_amd.layers.kv4 import KV4Cache
    starts = None if state["case"]["tokens"] == 1 else state["starts"]
    return KV4Cache(*state["cache"]).attend(0, state["q"], state["table"], state["lens"], starts)


def run(state):
    case = state["case"]
    if case["op"] == "cache_write":
        return _own_cache_write(state) if own else _plain_cache_write(state)
    if case["op"] == "cache_attend":
        return _own_cache_attend(state) if own else _plain_cache_attend(state)
    if case["op"] == "attention":
        out = _own_attention(state) if own else _plain_attention(state)
        if not case["train"]:
            return out
        grads = torch.autograd.grad(out, [state[n] for n in ("q", "k", "v")], state["grad"])
        return {"out": out.detach(), "d_q": grads[0], "d_k": grads[1], "d_v": grads[2]}
    out = _own_norm_rotary(state) if own else _plain_norm_rotary(state)
    if not case["train"]:
        return list(out)
    leaves = ("q", "k", "q_weight", "k_weight")
    grads = torch.autograd.grad(out, [state[n] for n in leaves], state["grads"])
    return {"out": [o.detach() for o in out], **{"d_" + n: g for n, g in zip(leaves, grads)}}


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm_rotary":
        cells = case["batch"] * case["len"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        # x -> y; trained: also dy -> dx (x is read once in a pass that did both)
        return {"bytes": cells * size * (4 if case["train"] else 2) + 8 * case["batch"] * case["len"] * case["axes"],
                "flops": cells * (20 if case["train"] else 8)}
    if case["op"] == "attention":
        seen = 0
        for n, m in zip(*_attention_lens(case)):   # key j of query i: j <= i + m - n
            full = min(n, m)                       # queries that see a key, the last of them all m
            seen += full * m - full * (full - 1) // 2
        lens, k_lens = (sum(x) for x in _attention_lens(case))
        cells, k_cells = lens * case["q_heads"] * case["dim"], k_lens * case["k_heads"] * case["dim"]
        # q, k, v -> out; trained: also d_out -> dq, dk, dv. Two products forward; five more backward
        return {"bytes": size * (cells * 4 + k_cells * 4 if case["train"] else cells * 2 + k_cells * 2),
                "flops": seen * case["q_heads"] * case["dim"] * 2 * (7 if case["train"] else 2)}
    held = case["k_heads"] * (case["dim"] // 2 + case["dim"] // 32) * 2   # bytes of a token's K and V
    if case["op"] == "cache_write":
        tokens = sum(_lengths(case, min(1, case["longest"])))
        cells = tokens * case["k_heads"] * case["dim"] * 2
        # k, v -> codes; the codes -> values
        return {"bytes": cells * (size + 2) + 2 * tokens * held, "flops": cells * 8}
    tokens, cells = sum(_lengths(case, case["tokens"])), case["seqs"] * case["tokens"] * case["q_heads"] * case["dim"]
    return {"bytes": tokens * held + 2 * size * cells, "flops": 4 * tokens * case["tokens"] * case["q_heads"] * case["dim"]}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_norm_rotary(state):
    case = state["case"]
    half, pos = case["rot"] // 2, state["pos"]
    which = torch.zeros(half, dtype=torch.long, device=pos.device) if state["axis"] is None else state["axis"].long()
    pos = pos[..., None] if state["axis"] is None else pos
    ang = pos[..., which].double() * state["freq"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=pos.device), ang)[:, :, None]
    first = torch.arange(half, device=pos.device)
    first, second = (2 * first, 2 * first + 1) if case["pairs"] == "interleaved" else (first, first + half)

    def turned(x, by):
        out = x.clone()
        z = torch.complex(x[..., first], x[..., second]) * by
        out[..., first], out[..., second] = z.real, z.imag
        return out

    out, back = [], {}
    for i, name in enumerate(("q", "k")):
        x, w = state[name].detach().double(), state[name + "_weight"].detach().double()
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + EPS)
        u = x * r
        out.append(turned(u * w, turn))
        if case["train"]:
            g = turned(state["grads"][i].double(), turn.conj())
            back["d_" + name + "_weight"] = (g * u).sum((0, 1, 2))
            g = g * w
            back["d_" + name] = r * (g - u * (g * u).mean(-1, keepdim=True))
    return {"out": out, **back} if case["train"] else out


def _attend64(q, k, v, offset, d_out=None):
    """Attention of q [H, L, D] over one head's k, v [M, D], query i seeing the keys up to i + offset; with d_out also the
    gradients of q, k and v."""
    n, m, c = q.shape[1], k.shape[0], q.shape[2] ** -0.5
    s = torch.matmul(q.reshape(-1, q.shape[2]), k.t().contiguous()).view(-1, n, m) * c
    see = torch.ones(n, m, dtype=torch.bool, device=q.device).tril(offset)
    s = torch.where(see, s, torch.full((), -math.inf, dtype=s.dtype, device=q.device))
    some = see.any(1)
    e = torch.exp(s - torch.where(some[:, None], s.max(-1, keepdim=True).values, torch.zeros_like(s[..., :1])))
    p = e / torch.where(some[:, None], e.sum(-1, keepdim=True), torch.ones_like(s[..., :1]))
    del s, e
    o = torch.matmul(p, v)
    if d_out is None:
        return o
    dp = torch.matmul(d_out, v.t().contiguous())
    ds = p * (dp - (d_out * o).sum(-1, keepdim=True)) * c
    return (o, torch.matmul(ds, k), torch.matmul(ds.transpose(1, 2).contiguous(), q).sum(0),
            torch.matmul(p.transpose(1, 2).contiguous(), d_out).sum(0))


def _exact_attention(state):
    case = state["case"]
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    out, grads = torch.zeros_like(q), [torch.zeros_like(x) for x in (q, k, v)]
    group = case["q_heads"] // case["k_heads"]
    at = k_at = 0
    for n, m in zip(*_attention_lens(case)):
        for h in range(case["k_heads"]):
            heads = slice(h * group, (h + 1) * group)
            one = (x.transpose(0, 1).contiguous() for x in (q[at:at + n, heads], k[k_at:k_at + m, h:h + 1], v[k_at:k_at + m, h:h + 1]))
            qh, (kh,), (vh,) = one
            if not m:
                continue
            if not case["train"]:
                out[at:at + n, heads] = _attend64(qh, kh, vh, m - n).transpose(0, 1)
                continue
            o, dq, dk, dv = _attend64(qh, kh, vh, m - n, state["grad"][at:at + n, heads].double().transpose(0, 1).contiguous())
            out[at:at + n, heads], grads[0][at:at + n, heads] = o.transpose(0, 1), dq.transpose(0, 1)
            grads[1][k_at:k_at + m, h], grads[2][k_at:k_at + m, h] = dk, dv
        at, k_at = at + n, k_at + m
    return {"out": out, "d_q": grads[0], "d_k": grads[1], "d_v": grads[2]} if case["train"] else out


def _decode64(code, scale):
    """sign, two exponent bits, one mantissa bit, times 2^(scale - 127)"""
    e, m = (code >> 1 & 3).double(), (code & 1).double()
    mag = torch.where(e > 0, (2 + m) * 2.0 ** (e - 2), m / 2)
    value = torch.where(code >> 3 > 0, -mag, mag)
    return (value.unflatten(-1, (-1, 32)) * 2.0 ** (scale.double()[..., None] - 127)).flatten(-2)


def _exact_cache_write(state):
    out = []
    for x in (state["k"], state["v"]):
        g = x.double().unflatten(-1, (-1, 32))
        top = g.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, -125)
        for s in range(-124, 127):   # (the least that will do)
            e = torch.where(top > 6 * 2.0 ** (s - 1), float(s), e)
        u = g / 2.0 ** e
        # the steps of e2m1: 1/2 below 2, 1 below 4, 2 above; torch rounds ties to even
        step = torch.where(u.abs() < 2, 0.5, torch.where(u.abs() < 4, 1.0, 2.0))
        out.append(((u / step).round() * step * 2.0 ** e).flatten(-2))
    return out


def _exact_cache_attend(state):
    case, n = state["case"], state["case"]["tokens"]
    q = state["q"].double().view(case["seqs"], n, case["k_heads"], -1, case["dim"])
    out = torch.zeros_like(q)
    for s, m in enumerate(_lengths(case, n)):
        pages = state["table"][s, :-(-m // PAGE)].long()
        k, v = (_decode64(c[pages].int(), e[pages].int()).transpose(0, 1).flatten(1, 2)[:, :m]
                for c, e in (state["codes"][:2], state["codes"][2:]))
        for h in range(case["k_heads"]):
            out[s, :, h] = _attend64(q[s, :, h].transpose(0, 1).contiguous(), k[h], v[h], m - n).transpose(0, 1)
    return out.view(state["q"].shape)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm_rotary": _exact_norm_rotary, "attention": _exact_attention, "cache_write": _exact_cache_write,
                "cache_attend": _exact_cache_attend}[case["op"]](state)
