"""The 64-bit definitions of causal self-attention: against differences, and the cache's format against its words."""
import pytest
import torch

from oracle import block, causal


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _differences(f, x, d, step=1e-6):
    """sum(f(x) d) differentiated by central differences, value by value."""
    out = torch.zeros_like(x)
    flat = x.view(-1)
    for i in range(flat.numel()):
        keep = flat[i].item()
        flat[i] = keep + step
        hi = (f() * d).sum()
        flat[i] = keep - step
        lo = (f() * d).sum()
        flat[i] = keep
        out.view(-1)[i] = (hi - lo) / (2 * step)
    return out


@pytest.mark.parametrize("n,m,causal_", [(4, 4, True), (3, 6, True), (6, 3, True), (3, 5, False), (1, 1, True)])
def test_attention_gradients_by_differences(n, m, causal_):
    g = _gen(n * m)
    q, k, v = (torch.randn(x, 3, dtype=torch.float64, generator=g) for x in (n, m, m))
    d = torch.randn(n, 3, dtype=torch.float64, generator=g)
    see = causal.visible(n, m, causal_, "cpu")
    r = causal.attend(q, k, v, see, 0.7, d)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        want = _differences(lambda: causal.attend(q, k, v, see, 0.7)["out"], x, d)
        assert (r[name] - want).abs().max() < 1e-7, name


def test_attention_shared_heads_add_up():
    g = _gen(1)
    q, k, v = torch.randn(7, 4, 8, generator=g), torch.randn(7, 2, 8, generator=g), torch.randn(7, 2, 8, generator=g)
    d = torch.randn(7, 4, 8, generator=g)
    r = causal.packed(q, k, v, [0, 3, 7], [0, 3, 7], d_out=d)
    ks, vs = (x.repeat_interleave(2, 1) for x in (k, v))
    full = causal.packed(q, ks, vs, [0, 3, 7], [0, 3, 7], d_out=d)
    assert torch.allclose(r["out"], full["out"])
    for name in ("dk", "dv"):
        assert torch.allclose(r[name], full[name].view(7, 2, 2, 8).sum(2))


@pytest.mark.parametrize("pairs", ["interleaved", "half"])
@pytest.mark.parametrize("dim,rot", [(8, 8), (8, 4), (7, 2)])
def test_norm_rotary_gradients_by_differences(dim, rot, pairs):
    g = _gen(dim + rot)
    x, d = (torch.randn(1, 3, 2, dim, dtype=torch.float64, generator=g) for _ in range(2))
    w = 1 + 0.3 * torch.randn(dim, dtype=torch.float64, generator=g)
    pos, freq = torch.tensor([[2, 5, 900]]), torch.linspace(0.1, 1, rot // 2, dtype=torch.float64)
    f = lambda: causal.norm_rotary(x, w, pos, freq, pairs=pairs, factor=1.2, eps=1e-3)[0][0]   # noqa: E731
    _, grads = causal.norm_rotary(x, w, pos, freq, pairs=pairs, factor=1.2, eps=1e-3, d=d)
    assert (grads["x"][0] - _differences(f, x, d)).abs().max() < 1e-7
    assert (grads["weight"][0] - _differences(f, w, d)).abs().max() < 1e-7


def test_encode_against_its_words():
    """The least power of two that leaves no magnitude over 6, the nearest code, ties to the even one."""
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    x = torch.zeros(1, 32)
    x[0, :12] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.0, -0.25, 0.26, 5.01])
    codes, scale = causal.encode(x)
    assert scale.item() == 127 and codes[0, :12].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 14, 8, 1, 7]
    for top, e in ((6.0, 0), (6.001, 1), (3.0, -1), (3.001, 0), (12.0, 1), (2.0 ** -140, -125), (0.0, -125)):
        x[0] = top
        assert causal.encode(x)[1].item() == e + 127, top
    g = _gen(3)
    y = torch.randn(50, 64, generator=g) * torch.exp2(torch.randint(-20, 20, (50, 1), generator=g).float())
    v = causal.values(*causal.encode(y))
    scale = 2.0 ** (causal.encode(y)[1].double() - 127).repeat_interleave(32, 1)
    steps = torch.tensor(grid, dtype=torch.float64)
    best = ((y.double().abs() / scale)[..., None] - steps).abs().amin(-1)
    assert torch.equal((v.abs() / scale - y.double().abs() / scale).abs(), best)
    x[0, 5] = float("nan")
    assert causal.encode(x)[1].item() == 255 and causal.values(*causal.encode(x)).isnan().all()


@pytest.mark.parametrize("d", [64, 128])
def test_pages_hold_what_was_put_there(d):
    """The layout read byte by byte: each code lands at one token and channel, and none is left out."""
    pages, heads = 2, 3
    g = _gen(d)
    k4 = torch.randint(0, 256, (pages, heads, 64, d // 2), generator=g, dtype=torch.uint8)
    v4 = torch.randint(0, 256, (pages, heads, 32 * d), generator=g, dtype=torch.uint8)
    ks = torch.randint(120, 130, (pages, heads, 64, d // 32), generator=g, dtype=torch.uint8)
    vs = torch.randint(120, 130, (pages, heads, 2 * d), generator=g, dtype=torch.uint8)
    k, v = causal.unpack_pages(k4, ks, v4, vs)
    for x, codes, scales in ((k, k4, ks), (v, v4, vs)):
        total = sum(causal.values((codes >> s & 15).long().view(-1, 1).expand(-1, 32), torch.full((codes.numel(), 1), 127))[:, 0].abs().sum()
                    for s in (0, 4))
        flat = causal.unpack_pages(k4, torch.full_like(ks, 127), v4, torch.full_like(vs, 127))[0 if x is k else 1]
        assert torch.equal(flat.abs().sum(), total)
        # the scales: one for each 32 channels of a token
        ratio = (x.abs().unflatten(-1, (-1, 32)).sum(-1) / flat.abs().unflatten(-1, (-1, 32)).sum(-1)).flatten().sort().values
        assert torch.equal(ratio, (2.0 ** (scales.double() - 127)).flatten().sort().values)


def test_cache_attend_is_attend_over_the_gathered_tokens():
    g = _gen(5)
    k, v = (torch.randn(4, 2, 64, 16, generator=g).double() for _ in range(2))
    q = torch.randn(3, 4, 16, generator=g)
    r = causal.cache_attend(q, k, v, [0, 2, 3], [70, 1], [[2, 0], [3, -1]])
    see = torch.ones(2, 70, dtype=torch.bool).tril(68)
    keys = torch.cat((k[2], k[0]), 1)[:, :70]
    vals = torch.cat((v[2], v[0]), 1)[:, :70]
    for h in range(4):
        assert torch.allclose(r["out"][:2, h], causal.attend(q[:2, h], keys[h // 2], vals[h // 2], see, 0.25)["out"])
        assert torch.equal(r["out"][2, h], v[3, h // 2, 0])


def test_rotation_of_the_definitions_agrees():
    x = torch.randn(1, 4, 2, 8, generator=_gen(6), dtype=torch.float64)
    freq = torch.linspace(0.1, 1, 4, dtype=torch.float64)
    pos = torch.arange(4)
    (y, _), _ = causal.norm_rotary(x, None, pos, freq, eps=0.0)
    r = x.square().mean(-1, keepdim=True).rsqrt()
    assert torch.allclose(y, block.rotary(x * r, pos, freq)[0])


@pytest.mark.parametrize("counts,lens", [([5], [130]), ([10, 2], [70, 64]), ([70, 3, 1], [128, 200, 129]), ([4], [0]), ([4, 9], [-3, 2])])
def test_cache_attend_sees_what_slots_hold(counts, lens):
    """A row sees the held tokens up to its own place, as write and read place them, also where a length passes the table."""
    g = _gen(sum(lens))
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    table = [[2 * i, 2 * i + 1] for i in range(len(counts))]
    table[0][0] = 90 if len(counts) > 1 else 0
    pages, rows = 2 * len(counts), starts[-1]
    k, v = (torch.randn(pages, 2, 64, 16, generator=g).double() for _ in range(2))
    q = torch.randn(rows, 4, 16, generator=g)
    out = causal.cache_attend(q, k, v, starts, lens, table)["out"]
    for s, n in enumerate(lens):
        held = causal.slots([0, max(n, 0)], [n], [table[s]], max(n, 0), pages)   # of each token of the sequence, where it lies
        for r in range(starts[s], starts[s + 1]):
            at = n - (starts[s + 1] - r)
            seen = [slot for slot in held[:max(at + 1, 0)] if slot is not None]
            for h in range(4):
                if not seen:
                    assert not out[r, h].any()
                    continue
                keys, vals = (torch.stack([x[p, h // 2, t] for p, t in seen]) for x in (k, v))
                p = torch.softmax(keys @ q[r, h].double() / 4, 0)
                assert torch.allclose(out[r, h], p @ vals)
