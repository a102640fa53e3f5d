"""Causal self-attention on the GPU against its definitions in 64 bits (oracle/causal.py).

Bounds, with h = half a step of the 16-bit type and e = 2^-24:
- Norm and rotation: h |y| + K e magnitude. A row's squares are added in 16 + 6 steps, halved by the root, with a dozen
  products around and the 12 roundings of a rotation: K = 36; its gradient has two such sums: K = 64. A weight's gradient
  adds a lane's rows (tokens * heads / (teams * workgroups), under 64 for the sizes here), up to 64 teams, 64 + 16 workgroups:
  K = 256.
- Attention: the weights are rounded to the type: h sum p |v|, then h |out|. fp32 work moves a weight by e times (D / 16 + 8)
  times the row's largest sum of |q| |k| (twice: its own logit and the row's sum), 64 for exponentials and the running
  sum's rescaling, and sums of L / 16 matrix products.
- Its gradients: dS is rounded too (h), and D = rowsum(dO o) is made of an output whose weights were rounded (h), and whose
  rest was (h^2). Elementwise these bounds are loose by the root of the keys, so the whole tensor's error is held too:
  roundings are independent, each of variance h^2 / 3 at most, and the sum of squared errors is allowed 4 times the sum of
  their variances.
"""
import pytest
import torch

from oracle import causal

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rand(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def _within(got, value, tol, what):
    assert got.shape == value.shape, what
    half = torch.finfo(got.dtype).eps / 2
    tol = tol + half * value.abs() + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double() - value).abs()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} of its bound (max error {err.max().item():.3e})"


def _together(got, value, variance, what):
    """The whole tensor's error: 4 times the variances of its roundings (the output's own among them)."""
    h2 = (torch.finfo(got.dtype).eps / 2) ** 2 / 3
    if got.numel() < 4096:
        return
    err, most = (got.double() - value).square().sum().item(), 4 * h2 * (variance.sum() + value.square().sum()).item()
    assert err <= most, f"{what}: squared error {err:.3e} of {most:.3e}"


# ---------------------------------------------------------------- norm and rotation


def _check_norm_rotary(seed, b, n, hq, hk, d, dtype="bf16", weight="same", layout="NHD", pairs="half", rot=None, axes=1, factor=1.0,
                       strided=False, train=True, wants=("q", "k", "q_weight", "k_weight"), pos=None, eps=1e-6):
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed
    g = _gen(seed)
    t = DT[dtype]
    shape = lambda h: (b, n, h, d) if layout == "NHD" else (b, h, n, d)   # noqa: E731

    def rows(h):
        if not strided:
            return _rand(g, *shape(h), std=1.7, dtype=t)
        return _rand(g, *shape(h)[:-1], d + 3, std=1.7, dtype=t)[..., 1:d + 1]

    q, k = rows(hq), rows(hk) if hk else None
    w = {}
    if weight != "none":
        wt = t if weight == "same" else torch.float32
        w = {"q_weight": _rand(g, d, std=0.4, mean=1.0, dtype=wt)}
        if hk:
            w["k_weight"] = _rand(g, d, std=0.4, mean=1.0, dtype=wt)
    rot = d - d % 2 if rot is None else rot
    if axes == 1:
        plan = Rotary.build(rot, DEV, pairs=pairs)
        pos = torch.randint(0, 100000, (b, n), generator=g, device=DEV) if pos is None else pos
    else:
        plan = Rotary.build(rot, DEV, pairs=pairs, sections=(rot // 2 - 2, 1, 1))
        pos = torch.randint(0, 5000, (b, n, 3), generator=g, device=DEV, dtype=torch.int32)
    plan.factor = factor
    leaves = {"q": q, "k": k, **w}
    leaves = {name: x.detach().requires_grad_(train and name in wants) for name, x in leaves.items() if x is not None}
    got = norm_rotary_embed(leaves["q"], leaves.get("k"), pos, plan, leaves.get("q_weight"), leaves.get("k_weight"), eps, layout)
    with torch.no_grad():
        again = norm_rotary_embed(leaves["q"], leaves.get("k"), pos, plan, leaves.get("q_weight"), leaves.get("k_weight"), eps, layout)
    nhd = (lambda x: x) if layout == "NHD" else (lambda x: x.transpose(1, 2))
    p64 = torch.arange(pos, pos + n, device=DEV) if isinstance(pos, int) else pos
    outs, ds, want = [], [], {}
    for i, name in enumerate(("q", "k")):
        if name not in leaves:
            assert got[i] is None
            continue
        x = leaves[name]
        assert got[i].dtype == t and got[i].shape == x.shape and got[i].is_contiguous() and torch.equal(got[i], again[i])
        dy = _rand(g, *x.shape, dtype=t)
        (y, mag), grads = causal.norm_rotary(nhd(x), w.get(name + "_weight"), p64, plan.freq, plan.axis, pairs, factor, eps, nhd(dy))
        what = f"{name} {b}x{n}x{x.shape} {dtype}"
        _within(nhd(got[i].detach()), y, 36 * E * mag, what)
        want[name], want[name + "_weight"] = [nhd(z) for z in grads["x"]], grads["weight"]
        outs.append(got[i])
        ds.append(dy)
    if not train:
        return
    names = [m for m in leaves if leaves[m].requires_grad]
    for name, dx in zip(names, torch.autograd.grad(outs, [leaves[m] for m in names], ds)):
        value, mag = want[name]
        assert dx.dtype == leaves[name].dtype and dx.shape == leaves[name].shape
        _within(dx, value, (64 if name in ("q", "k") else 256) * E * mag, f"d_{name} {b}x{n} heads {hq} {hk} of {d} {dtype}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (64, 64), (80, 80), (96, 24), (256, 256), (2, 2), (6, 4), (250, 250), (129, 2),
                                   (512, 512), (511, 300), (508, 4), (40, 12)])
@pytest.mark.parametrize("pairs", ["interleaved", "half"])
def test_norm_rotary_head_sizes(d, rot, pairs, dtype):
    _check_norm_rotary(d + rot, 2, 7, 3, 2, d, dtype, rot=rot, pairs=pairs)


@pytest.mark.parametrize("b,n,hq,hk", [(1, 1, 1, 1), (1, 1, 1, 0), (3, 1, 14, 2), (1, 2100, 5, 1), (2, 515, 12, 12), (1, 9, 40, 8), (5, 3, 1, 7)])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_norm_rotary_sizes(b, n, hq, hk, layout):
    _check_norm_rotary(n + hq, b, n, hq, hk, 128, layout=layout)
    _check_norm_rotary(n + hq, b, n, hq, hk, 64, "fp16", "fp32", layout, "interleaved", axes=3)


@pytest.mark.parametrize("weight", ["none", "same", "fp32"])
@pytest.mark.parametrize("strided", [False, True])
def test_norm_rotary_forms(weight, strided):
    for dtype in DT:
        _check_norm_rotary(5, 2, 33, 4, 2, 128, dtype, weight, strided=strided, factor=1.3, eps=1e-5)
        _check_norm_rotary(6, 1, 33, 4, 2, 72, dtype, weight, strided=strided, rot=40, pos=12345)


@pytest.mark.parametrize("wants", [("q",), ("k",), ("q_weight",), ("k_weight",), ("q", "k_weight"), ("k", "q_weight"), ("q_weight", "k_weight")])
def test_norm_rotary_single_gradients(wants):
    _check_norm_rotary(8, 2, 65, 6, 3, 128, wants=wants)


def test_norm_rotary_one_output_s_gradient():
    """The gradient of one output alone: the other input's is zero."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed
    g = _gen(9)
    q, k = (_rand(g, 1, 40, h, 128, dtype=torch.bfloat16).requires_grad_() for h in (4, 2))
    w = _rand(g, 128, mean=1.0).requires_grad_()
    plan = Rotary.build(128, DEV)
    oq, ok = norm_rotary_embed(q, k, 3, plan, w, w)
    d = _rand(g, *ok.shape, dtype=torch.bfloat16)
    dq, dk, dw = torch.autograd.grad(ok, (q, k, w), d, allow_unused=True)
    assert dq is None or not dq.any()
    _, grads = causal.norm_rotary(k, w, torch.arange(3, 43, device=DEV), plan.freq, d=d)
    _within(dk, grads["x"][0], 64 * E * grads["x"][1], "dk")
    _within(dw, grads["weight"][0], 256 * E * grads["weight"][1], "dw")


def test_norm_rotary_rows_of_zeros_and_nan():
    """A row of zeros stays zero (eps); a NaN or an infinity stays in its own row."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed
    x = _rand(_gen(10), 1, 6, 3, 128, dtype=torch.bfloat16)
    x[0, 1, 2] = 0
    x[0, 2, 0, 5] = float("nan")
    x[0, 3, 1, 7] = float("inf")
    plan = Rotary.build(128, DEV)
    y = norm_rotary_embed(x, None, 0, plan)[0]
    bad = torch.zeros(6, 3, dtype=torch.bool, device=DEV)
    bad[2, 0] = bad[3, 1] = True
    assert bool(y[0][~bad].isfinite().all()) and not y[0, 1, 2].any() and bool(y[0, 2, 0].isnan().all())
    assert not y[0, 3, 1].isfinite().all()


# ---------------------------------------------------------------- packed attention


def _starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _packed_bounds(r, keys, d, dtype):
    """What fp32 work may move, relative to the parts of the bound."""
    return E * (keys / 16 + 64 + 2 * (d / 16 + 8) * r["logit"])


def _check_packed(seed, lens, k_lens, hq, hk, d, dtype="bf16", train=True, causal_=True, scale=None, tail=0, head=0, rows=None, d_rows=None,
                  std=1.0, mean=0.3, grad_std=1.0):
    from lingbot_world_v2_realtime_amd import packed_attention
    g = _gen(seed)
    t = DT[dtype]
    st, ks = _starts(lens, head), _starts(k_lens, head)
    make = rows or (lambda n, h: _rand(g, n, h, d, std=std, dtype=t))
    q, k, v = make(st[-1] + tail, hq), make(ks[-1] + tail, hk), make(ks[-1] + tail, hk)
    if rows is None and k.numel():
        k += _rand(g, hk, d, std=mean, dtype=t)
    q, k, v = (x.detach().requires_grad_(train) for x in (q, k, v))
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    args = (dev(st), None if st == ks and q.shape[0] == k.shape[0] else dev(ks), scale, causal_)
    out = packed_attention(q, k, v, *args)
    with torch.no_grad():
        assert torch.equal(out, packed_attention(q, k, v, *args))
    do = (d_rows or (lambda n, h: _rand(g, n, h, d, std=grad_std, dtype=t)))(q.shape[0], hq)
    r = causal.packed(q.detach(), k.detach(), v.detach(), st, ks, scale, causal_, do if train else None)
    what = f"{lens} / {k_lens}, heads {hq} {hk} of {d}, {dtype}"
    assert out.dtype == t and out.is_contiguous()
    if "out" not in r:
        assert not out.any()
        return out
    h = torch.finfo(t).eps / 2
    keys = max(k_lens)
    rel = _packed_bounds(r, keys, d, dtype)
    _within(out.detach(), r["out"], (h + rel) * r["p_v"] + keys * 2.0 ** -35, what)
    _together(out.detach(), r["out"], r["p2_v2"], what)
    if not train:
        return out
    grads = torch.autograd.grad(out, (q, k, v), do)
    again = torch.autograd.grad(packed_attention(q, k, v, *args), (q, k, v), do)
    top = rel.max()
    group = hq // hk
    for name, x, y in zip(("dq", "dk", "dv"), grads, again):
        assert x.dtype == t and torch.equal(x, y), f"{what}: {name}"
        steps = E * ((keys if name == "dq" else max(lens) * group) / 16 + 16)
        tol = (h + steps) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (top + h * h + E * (d / 16 + 8)) * r[name + "_wide32"]
        # (the smallest numbers of fp16 are a fixed step apart, of weights raised by 2^10 and of dS brought near 1)
        _within(x, r[name], tol, f"{what}: {name}")
        _together(x, r[name], r[name + "_sq"] + r.get(name + "_d2", 0), f"{what}: {name}")
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257, 400])
def test_packed_one_sequence(n, d, dtype):
    _check_packed(n, [n], [n], 2, 1, d, dtype)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (8, 2), (12, 4), (24, 3), (5, 1), (16, 1)])
def test_packed_heads(hq, hk):
    _check_packed(hq, [70, 1, 0, 133], [70, 1, 0, 133], hq, hk, 128)
    _check_packed(hq, [70, 1, 0, 133], [70, 1, 0, 133], hq, hk, 64, "fp16")


@pytest.mark.parametrize("causal_", [True, False])
@pytest.mark.parametrize("lens,k_lens", [([40, 3, 0, 129], [140, 3, 70, 200]), ([130, 70, 5], [60, 70, 0]), ([200, 64], [1, 63]),
                                         ([1, 1, 1], [300, 64, 65]), ([0, 0], [5, 0]), ([64, 64], [0, 0]), ([90, 64], [64, 90])])
def test_packed_lengths_of_keys(lens, k_lens, causal_):
    """A prefix in the keys alone, fewer keys than queries (rows that see nothing), none at all."""
    _check_packed(11, lens, k_lens, 4, 2, 128, causal_=causal_, tail=3, head=2)
    _check_packed(12, lens, k_lens, 4, 2, 64, "fp16", causal_=causal_, tail=130, head=70)


def test_packed_rows_of_no_sequence():
    """Rows before the first sequence and behind the last, whatever they hold: 0, and no gradient; they reach no other row."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g = _gen(13)
    for d in (64, 128):
        q, k, v = (_rand(g, 300, h, d, dtype=torch.bfloat16) for h in (4, 2, 2))
        starts = torch.tensor([37, 90, 90, 201], dtype=torch.int32, device=DEV)
        want = packed_attention(q, k, v, starts)
        outside = torch.ones(300, dtype=torch.bool, device=DEV)
        outside[37:201] = False
        for odd in (float("nan"), float("inf")):
            x, y, z = (t.clone() for t in (q, k, v))
            for t in (x, y, z):
                t[outside] = odd
                t.requires_grad_()
            out = packed_attention(x, y, z, starts)
            assert torch.equal(out, want) and not out[outside].any()
            do = torch.full_like(out, odd)
            do[~outside] = _rand(_gen(14), 164, 4, d, dtype=torch.bfloat16)
            for grad in torch.autograd.grad(out, (x, y, z), do):
                assert not grad[outside].any() and bool(grad.isfinite().all())


@pytest.mark.parametrize("seqs", [64, 65, 130, 4200])
def test_packed_many_sequences(seqs):
    lens = [(5 * i) % 4 for i in range(seqs)]
    if seqs > 1000:   # (the definition takes its time)
        lens = [n if i % 97 == 0 else 0 for i, n in enumerate(lens)]
    lens[-1] = 40
    _check_packed(seqs, lens, lens, 2, 2, 64)


def test_packed_strides():
    """Parts of one projection, rows of a batch's padding, views that the kernels do not load from (copied)."""
    g = _gen(15)

    def fused(n, h):
        return _rand(g, n, 3 * h, 128, dtype=torch.bfloat16)[:, h:2 * h]

    def odd(n, h):
        return _rand(g, n, h, 131, dtype=torch.bfloat16)[..., 1:129]

    def turned(n, h):
        return _rand(g, h, n, 128, dtype=torch.bfloat16).transpose(0, 1)

    def spread(n, h):
        return _rand(g, n, 1, 128, dtype=torch.bfloat16).expand(n, h, 128)

    for rows in (fused, odd, turned, spread):
        _check_packed(16, [70, 130], [70, 130], 4, 2, 128, rows=rows, d_rows=rows)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_packed_peaked_and_flat(dtype):
    """Logits in the hundreds (one key takes all) and all alike; a scale of its own."""
    _check_packed(17, [200], [200], 2, 2, 128, dtype, std=6.0, mean=0.0)
    _check_packed(18, [333], [333], 2, 2, 64, dtype, scale=1e-4)
    _check_packed(19, [150], [150], 2, 1, 128, dtype, scale=0.7)


@pytest.mark.parametrize("grad_std", [1e-6, 1e-3, 3000.0])
def test_packed_gradients_small_and_large(grad_std):
    """Gradients that a loss's scale made very small or large: dS leaves fp16's range where the gradients do not."""
    for d in (64, 128):
        _check_packed(20, [300, 65], [300, 65], 4, 2, d, "bf16", grad_std=grad_std)
        if grad_std >= 1e-3:
            # (dO itself keeps its digits down to 2^-14)
            _check_packed(21, [300, 65], [300, 65], 4, 2, d, "fp16", grad_std=grad_std, std=0.5 if grad_std > 1 else 1.0)


def test_packed_long_rows():
    _check_packed(22, [1000, 1508], [1000, 1508], 2, 1, 128)
    _check_packed(23, [17], [6032], 2, 1, 128, train=False)
    _check_packed(24, [2100], [2100], 2, 2, 64, "fp16")


def test_packed_single_gradients():
    from lingbot_world_v2_realtime_amd import packed_attention
    g = _gen(25)
    starts = torch.tensor([0, 100, 180], dtype=torch.int32, device=DEV)
    base = [_rand(g, 180, h, 128, dtype=torch.bfloat16) for h in (4, 2, 2)]
    do = _rand(g, 180, 4, 128, dtype=torch.bfloat16)
    full = torch.autograd.grad(packed_attention(*(x.requires_grad_() for x in base), starts), base, do)
    for i in range(3):
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate(base)]
        (got,) = torch.autograd.grad(packed_attention(*leaves, starts), [leaves[i]], do)
        assert torch.equal(got, full[i])


def test_packed_wrong_starts_stay_inside():
    """Starts past the tensor are cut at its end, below zero at its start; what lies in the sequences is right."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g = _gen(26)
    q, k, v = (_rand(g, 100, 2, 64, dtype=torch.bfloat16) for _ in range(3))
    dev = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    assert torch.equal(packed_attention(q, k, v, dev(-5, 40, 1000)), packed_attention(q, k, v, dev(0, 40, 100)))
    packed_attention(q, k, v, dev(0, 80, 20, 2 ** 31 - 1))   # falling starts: no particular answer


# ---------------------------------------------------------------- the cache


def _lists(*ts):
    return [t.tolist() for t in ts]


def _table(g, counts, pages, width=None):
    """Distinct pages for each sequence, -1 behind."""
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    width = width or max(max(counts), 1)
    return [[order.pop() for _ in range(n)] + [-1] * (width - n) for n in counts]


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_cache_write_and_read(heads, d, dtype):
    from lingbot_world_v2_realtime_amd import KV4Cache
    g = _gen(heads + d)
    new, lens = [0, 1, 130, 64, 7], [5, 64, 190, 64, 71]
    st, pages = _starts(new, 2), 12
    rows = st[-1] + 4
    table = _table(g, [-(-n // 64) for n in lens], pages, 4)
    k = _rand(g, rows, heads, d, dtype=DT[dtype]) * torch.exp2(torch.randint(-12, 12, (rows, heads, 1), generator=g, device=DEV)).to(DT[dtype])
    v = _rand(g, rows, heads, d, std=3.0, dtype=DT[dtype])
    k[5], v[7, 0, 33] = 0, 0.0
    cache = KV4Cache.empty(2, pages, heads, d, DEV)
    cache.write(1, k, v, _dev(table), _dev(lens), _dev(st))
    at = causal.slots(st, lens, table, rows, pages)
    pk, pv = causal.unpack_pages(cache.k[1], cache.k_scale[1], cache.v[1], cache.v_scale[1])
    written = torch.zeros(pages, 64, dtype=torch.bool)
    rk, rv = cache.read(1, _dev(table), _dev(lens), _dev(st), tokens=rows)
    assert rk.dtype == torch.bfloat16 and rk.shape == k.shape
    for x, pagev, r in ((k, pk, rk), (v, pv, rv)):
        want = causal.values(*causal.encode(x))
        for i, slot in enumerate(at):
            if slot is None:
                assert not r[i].any()
                continue
            written[slot] = True
            assert torch.equal(pagev[slot[0], :, slot[1]], want[i]), (i, slot)
            assert torch.equal(r[i].double(), want[i]), (i, slot)
    free = (~written).to(DEV)
    for pagev in (pk, pv):   # nothing else was touched
        assert not pagev.transpose(1, 2)[free].any()
    assert not any(x[0].any() for x in (cache.k, cache.k_scale, cache.v, cache.v_scale))


def test_cache_holds_every_value():
    """Every finite bf16 value as a group's largest, and next to it: the scale's choice, ties, the least scale, the largest."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    bits = torch.arange(0, 0x7F80, device=DEV, dtype=torch.int32)
    top = bits.to(torch.int16).view(torch.bfloat16)
    x = top[:, None] * torch.linspace(-1, 1, 32, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = top
    rows = -(-x.shape[0] // 4)
    k = torch.zeros(rows * 4, 32, dtype=torch.bfloat16, device=DEV)
    k[:x.shape[0]] = x
    k = k.view(rows, 1, 128)
    v = -k.flip(0).contiguous()
    pages = -(-rows // 64)
    cache = KV4Cache.empty(1, pages, 1, 128, DEV)
    table, lens, st = _dev([list(range(pages))]), _dev([rows]), _dev([0, rows])
    cache.write(0, k, v, table, lens, st)
    for x, r in zip((k, v), cache.read(0, table, lens, st, tokens=rows)):
        assert torch.equal(r.double(), causal.values(*causal.encode(x)))


def test_cache_values_that_are_not_finite():
    """A group with a NaN or an infinity is NaN, the groups beside it are not."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    for dtype in (torch.bfloat16, torch.float16):
        k, v = (_rand(_gen(30 + i), 3, 2, 128, dtype=dtype) for i in range(2))
        k[0, 1, 40], k[1, 0, 3], v[2, 1, 127] = float("nan"), float("inf"), -float("inf")
        cache = KV4Cache.empty(1, 2, 2, 128, DEV)
        table, lens, st = _dev([[1]]), _dev([3]), _dev([0, 3])
        cache.write(0, k, v, table, lens, st)
        for x, r in zip((k, v), cache.read(0, table, lens, st, tokens=3)):
            bad = (~x.isfinite()).unflatten(-1, (-1, 32)).any(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2)
            assert torch.equal(r.isnan(), bad)
            assert torch.equal(r.double()[~bad], causal.values(*causal.encode(x))[~bad])


def _filled(g, pages, heads, d):
    """A cache whose every byte is something: random codes, scales around 1."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    c = KV4Cache.empty(1, pages, heads, d, DEV)
    for x in (c.k, c.v):
        x.copy_(torch.randint(0, 256, x.shape, generator=g, device=DEV, dtype=torch.uint8))
    for x in (c.k_scale, c.v_scale):
        x.copy_(torch.randint(124, 128, x.shape, generator=g, device=DEV, dtype=torch.uint8))
    return c


def _check_cache_attend(seed, counts, lens, hq, hk, d, dtype="bf16", width=None, head=0, tail=0, scale=None, starts=True, bad=None, std=1.0):
    g = _gen(seed)
    t = DT[dtype]
    st = _starts(counts, head)
    pages = sum(-(-max(n, 0) // 64) for n in lens) + 2
    cache = _filled(g, pages, hk, d)
    table = _table(g, [-(-max(n, 0) // 64) for n in lens], pages, width)
    if bad:
        bad(table)
    q = _rand(g, st[-1] + tail, hq, d, std=std, dtype=t)
    kv = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    out = cache.attend(0, q, _dev(table), _dev(lens), _dev(st) if starts else None, scale)
    assert out.dtype == t and out.shape == q.shape
    assert torch.equal(out, cache.attend(0, q, _dev(table), _dev(lens), _dev(st) if starts else None, scale))
    r = causal.cache_attend(q, *kv, st, lens, table, scale)
    what = f"{counts} of {lens}, heads {hq} {hk} of {d}, {dtype}"
    # weights of bf16, or of twice its length
    h = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -16
    rel = _packed_bounds(r, max(max(lens), 1), d, dtype)
    _within(out, r["out"], (h + rel) * r["p_v"], what)
    _together(out, r["out"], r["p2_v2"], what)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 5000])
def test_cache_attend_lengths(n, d, dtype):
    _check_cache_attend(n, [1], [n], 4, 2, d, dtype, starts=False)


@pytest.mark.parametrize("hq,hk", [(1, 1), (12, 12), (12, 4), (32, 8), (16, 1), (17, 1), (40, 1), (96, 1), (150, 2)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_cache_attend_heads(hq, hk, dtype):
    _check_cache_attend(hq, [1, 1, 1], [200, 0, 77], hq, hk, 128, dtype, starts=False)
    _check_cache_attend(hq, [3, 0, 2], [200, 5, 77], hq, hk, 64, dtype, head=1, tail=2)


@pytest.mark.parametrize("counts,lens", [([5, 5, 5], [5, 700, 66]), ([16, 1, 0, 7], [300, 1, 9, 129]), ([70], [130]), ([9, 4], [3, 4]), ([1, 2], [0, 1]),
                                         ([40] * 3, [40, 41, 2000])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_cache_attend_several_tokens(counts, lens, dtype):
    """A sequence's newest tokens see each other causally; where the cache holds fewer than the call has, the first see nothing."""
    _check_cache_attend(41, counts, lens, 8, 2, 128, dtype, head=3, tail=1)
    _check_cache_attend(42, counts, lens, 3, 3, 64, dtype)


def test_cache_attend_many_sequences():
    lens = [(37 * i) % 150 for i in range(200)]
    _check_cache_attend(43, [1] * 200, lens, 4, 2, 64, starts=False)
    _check_cache_attend(44, [i % 3 for i in range(200)], lens, 4, 2, 64)


def test_cache_attend_wide_tables_and_bad_pages():
    """A table wider than the sequences (rows of it are -1 past them), pages that are not there: their tokens are not seen; lengths past
    the table are cut."""
    _check_cache_attend(45, [1, 2], [100, 260], 4, 2, 128, width=300)

    def bad(table):
        table[0][1], table[1][0], table[1][3] = -1, 10 ** 6, -(2 ** 31)

    _check_cache_attend(46, [1, 2], [200, 260], 4, 2, 128, bad=bad)
    _check_cache_attend(47, [1, 2], [200, 260], 4, 2, 64, "fp16", bad=bad, width=90)

    def none(table):
        table[0][:] = [-1] * len(table[0])

    _check_cache_attend(48, [1, 2], [100, 260], 4, 2, 128, bad=none)


def test_cache_attend_peaked():
    for dtype in ("bf16", "fp16"):
        _check_cache_attend(49, [2, 1], [700, 300], 4, 2, 128, dtype, std=8.0)
        _check_cache_attend(50, [2, 1], [700, 300], 4, 2, 128, dtype, scale=1e-3)


def test_cache_attend_does_not_see_what_it_should_not():
    """NaN in tokens behind the last, in pages of nobody, and in a token that later rows alone see."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        g = _gen(51)
        c = _filled(g, 6, 2, d)
        table, lens, st = [[4, 2, 0], [1, -1, -1]], [150, 40], [0, 6, 7]
        q = _rand(g, 7, 6, d, dtype=dtype)
        args = (_dev(table), _dev(lens), _dev(st))
        want = c.attend(0, q, *args)
        ok = {(4, i) for i in range(64)} | {(2, i) for i in range(64)} | {(0, i) for i in range(22)} | {(1, i) for i in range(40)}
        odd = KV4Cache(*(x.clone() for x in (c.k, c.k_scale, c.v, c.v_scale)))
        mark = torch.zeros(6, 64, dtype=torch.bool)
        for p in range(6):
            for i in range(64):
                mark[p, i] = (p, i) not in ok

        def poison(cache, mark):
            cache.k_scale[0][mark[:, None, :, None].expand(cache.k_scale[0].shape)] = 255
            for p, t in mark.nonzero().tolist():
                for grp in range(d // 32):
                    cache.v_scale[0, p, :, (((t // 32) * 4 + (t >> 2 & 3)) * (d // 32) + grp) * 8 + (t >> 4 & 1) * 4 + (t & 3)] = 255

        poison(odd, mark.to(DEV))
        assert torch.equal(odd.attend(0, q, *args), want)
        # token 147 of the first sequence (page 0, place 19) is seen by its rows 3, 4 and 5
        mark.zero_()
        mark[0, 19] = True
        poison(odd, mark.to(DEV))
        got = odd.attend(0, q, *args)
        seen = torch.tensor([0, 0, 0, 1, 1, 1, 0], dtype=torch.bool, device=DEV)
        assert torch.equal(got[~seen], want[~seen]) and bool(got[seen].isnan().all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_norm_rotary_weights_of_a_larger_buffer(dtype):
    """Weights that lie anywhere in a flat buffer, and their gradients."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed
    g = _gen(60)
    flat = _rand(g, 300, mean=1.0, dtype=DT[dtype]).requires_grad_()
    q = _rand(g, 1, 9, 4, 128, dtype=torch.bfloat16)
    plan, dy = Rotary.build(128, DEV), _rand(g, 1, 9, 4, 128, dtype=torch.bfloat16)
    for at in (1, 3, 8):
        out = norm_rotary_embed(q, q, 5, plan, flat[at:at + 128], flat[at + 128:at + 256])
        (got,) = torch.autograd.grad(out, flat, (dy, dy))
        for i in range(2):
            part = slice(at + 128 * i, at + 128 * i + 128)
            (y, mag), grads = causal.norm_rotary(q, flat[part], torch.arange(5, 14, device=DEV), plan.freq, d=dy)
            _within(out[i].detach(), y, 36 * E * mag, f"at {at}")
            _within(got[part], grads["weight"][0], 256 * E * grads["weight"][1], f"dw at {at}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,lens", [([200], [200]), ([97], [161]), ([33, 0, 64, 31], [40, 7, 96, 95]), ([500, 3, 160], [10, 3, 161]),
                                      ([64, 64], [64, 63]), ([32, 96], [0, 5000])])
def test_cache_write_and_read_blocks(new, lens, d):
    """Prompts: blocks of 32 tokens, whole and cut, tokens before the first and past the table, what lies beside them untouched."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    g = _gen(sum(new) + d)
    heads, pages = 3, 16
    st, rows = _starts(new, 3), 3 + sum(new) + 5
    table = _table(g, [min(4, -(-n // 64)) for n in lens], pages, 4)
    table[0][1] = 77
    k, v = (_rand(g, rows, heads, d, std=2.0, dtype=torch.bfloat16) for _ in range(2))
    cache = _filled(g, pages, heads, d)
    before = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    args = (_dev(table), _dev(lens), _dev(st))
    cache.write(0, k, v, *args)
    at = causal.slots(st, lens, table, rows, pages)
    after = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    got = cache.read(0, *args, tokens=rows)
    for x, old, now, r in zip((k, v), before, after, got):
        value = causal.values(*causal.encode(x))
        for i, slot in enumerate(at):
            if slot is None:
                assert not r[i].any(), i
            else:
                old[slot[0], :, slot[1]] = value[i]
                assert torch.equal(r[i].double(), value[i]), i
        assert torch.equal(old, now)
