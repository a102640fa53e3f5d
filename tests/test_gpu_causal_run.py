"""Causal self-attention on the GPU as it is used: norm and rotation, packed attention, the cache and the attention that reads it
one after the other; in graphs, on several streams, with values that are not finite where nothing sees them, and in tensors of
more than 2^31 bytes. Bounds as in test_gpu_causal.py.
"""
import pytest
import torch

from oracle import causal
from test_gpu_causal import DEV, DT, E, _check_cache_attend, _check_norm_rotary, _check_packed, _dev, _filled, _gen, _packed_bounds, _rand, _starts, _table, _within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("hq,hk,d,dtype", [(8, 2, 128, "bf16"), (6, 6, 64, "fp16")])
def test_prompts_then_tokens(hq, hk, d, dtype):
    """Prompts through norm, rotation and packed attention into the cache, then tokens one by one and a few drafted ones: each
    against 64 bits of what the cache holds; read() with packed_attention gives the rows that attend() gives."""
    from lingbot_world_v2_realtime_amd import KV4Cache, Rotary, norm_rotary_embed, packed_attention
    g, t = _gen(hq + d), DT[dtype]
    plan = Rotary.build(d, DEV, pairs="half")
    qw, kw = (_rand(g, d, std=0.2, mean=1.0, dtype=t) for _ in range(2))
    lens = [130, 1, 70, 64]
    seqs, pages = len(lens), 16
    table = _table(g, [4, 2, 3, 2], pages, 4)
    cache = KV4Cache.empty(3, pages, hk, d, DEV)
    layer = 2
    steps = [lens, [1] * seqs, [1] * seqs, [3, 0, 2, 1], [1] * seqs]
    held = [0] * seqs
    for i, new in enumerate(steps):
        held = [a + b for a, b in zip(held, new)]
        st, rows = _starts(new), sum(new)
        pos = torch.cat([torch.arange(n - c, n) for n, c in zip(held, new)]).to(DEV)
        q, k, v = _rand(g, 1, rows, hq, d, dtype=t), _rand(g, 1, rows, hk, d, dtype=t), _rand(g, rows, hk, d, dtype=t)
        qr, kr = norm_rotary_embed(q, k, pos, plan, qw, kw)
        for x, w, y in ((q, qw, qr), (k, kw, kr)):
            (want, mag), _ = causal.norm_rotary(x, w, pos, plan.freq, pairs="half")
            _within(y, want, 36 * E * mag, f"step {i}")
        one = [1] * seqs == new
        args = (_dev(table), _dev(held), None if one else _dev(st))
        cache.write(layer, kr[0], v, *args)
        kv = causal.unpack_pages(cache.k[layer], cache.k_scale[layer], cache.v[layer], cache.v_scale[layer])
        for j, (s, c) in enumerate((s, c) for s, n in enumerate(new) for c in range(n)):
            at = held[s] - new[s] + c
            for page, x in zip(kv, (kr[0], v)):
                assert torch.equal(page[table[s][at // 64], :, at % 64], causal.values(*causal.encode(x[j])))
        h = torch.finfo(t).eps / 2
        if i == 0:   # the prompts attend their own keys, as they are
            out = packed_attention(qr[0], kr[0], v, args[2])
            r = causal.packed(qr[0], kr[0], v, st, st)
            _within(out, r["out"], (h + _packed_bounds(r, max(lens), d, dtype)) * r["p_v"] + max(lens) * 2.0 ** -35, "prompts")
        out = cache.attend(layer, qr[0], *args)
        r = causal.cache_attend(qr[0], *kv, st, held, table)
        rel = _packed_bounds(r, max(held), d, dtype)
        _within(out, r["out"], (2.0 ** -8 if dtype == "bf16" else 2.0 ** -16) * r["p_v"] + rel * r["p_v"], f"step {i}")
        full = _starts(held)
        rk, rv = cache.read(layer, args[0], args[1], _dev(full), tokens=full[-1])
        again = packed_attention(qr[0], rk.to(t), rv.to(t), _dev(st), _dev(full))
        _within(again, r["out"], (h + rel) * r["p_v"] + max(held) * 2.0 ** -35, f"step {i}, read and packed")


def test_training_step_together():
    """A training step's norm, rotation and attention: the gradients of x's q and k rows and of the weights, against the formulas
    one behind the other (the bounds of the two: attention's error goes on through the norm's gradient, |r (1 + u mean(u))| wide)."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    g = _gen(3)
    lens, hq, hk, d = [70, 1, 129], 4, 2, 64
    st, plan = _starts(lens), Rotary.build(d, DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    q, k, v = (_rand(g, 1, sum(lens), h, d, dtype=torch.bfloat16).requires_grad_() for h in (hq, hk, hk))
    qw, kw = (_rand(g, d, std=0.2, mean=1.0).requires_grad_() for _ in range(2))
    do = _rand(g, sum(lens), hq, d, dtype=torch.bfloat16)
    qr, kr = norm_rotary_embed(q, k, pos, plan, qw, kw)
    qr.retain_grad()
    kr.retain_grad()
    packed_attention(qr[0], kr[0], v[0], _dev(st)).backward(do)
    r = causal.packed(qr[0].detach(), kr[0].detach(), v[0].detach(), st, st, d_out=do)
    for x, w, y, name in ((q, qw, qr, "dq"), (k, kw, kr, "dk")):
        assert (y.grad[0].double() - r[name]).square().sum() <= 2.0 ** -14 * r[name].square().sum(), name   # (1 / 128 of it)
        _, grads = causal.norm_rotary(x, w, pos, plan.freq, d=y.grad)
        _within(x.grad, grads["x"][0], 64 * E * grads["x"][1], name)
        _within(w.grad, grads["weight"][0], 256 * E * grads["weight"][1], name + " weight")
    assert (v.grad[0].double() - r["dv"]).square().sum() <= 2.0 ** -14 * r["dv"].square().sum()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gradients_against_differences(dtype):
    """The loss's change along a direction, in 64 bits at the rounded inputs, against the gradients' product with it. A gradient
    of n values, each rounded (h of itself, and of what is added in it as much again), moves the product by the root of their
    squares; the difference itself is off by step^2."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    g, t = _gen(12), DT[dtype]
    lens, d = [40, 25], 64
    st, plan, pos = _starts(lens), Rotary.build(d, DEV), torch.cat([torch.arange(n) for n in lens]).to(DEV)
    q, k, v = (_rand(g, sum(lens), h, d, dtype=t).requires_grad_() for h in (4, 2, 2))
    w = _rand(g, d, std=0.2, mean=1.0).requires_grad_()
    do = _rand(g, sum(lens), 4, d, dtype=t)
    qr, _ = norm_rotary_embed(q[None], None, pos, plan, w)
    grads = torch.autograd.grad(packed_attention(qr[0], k, v, _dev(st)), (q, k, v, w), do)

    def loss(q, k, v, w):
        (y, _), _ = causal.norm_rotary(q[None], w, pos, plan.freq)
        return (causal.packed(y[0], k, v, st, st)["out"] * do.double()).sum()

    leaves = [x.detach().double() for x in (q, k, v, w)]
    for i, got in enumerate(grads):
        step = torch.randn(got.shape, generator=g, device=DEV, dtype=torch.float64)
        at = lambda e: loss(*[x + e * step if j == i else x for j, x in enumerate(leaves)])   # noqa: E731
        e = 1e-4
        diff = (at(e) - at(-e)) / (2 * e)
        most = 16 * torch.finfo(t).eps * (got.double() * step).norm() + 1e-6 * step.norm()
        # (the rotated q is rounded before the attention sees it: a change of the loss's gradient of h, as much again)
        assert abs((got.double() * step).sum() - diff) <= most, ("q", "k", "v", "weight")[i]


# ---------------------------------------------------------------- graphs and streams


def _captured(fn):
    """fn captured, after a run on a side stream."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_serving_in_a_graph():
    """One captured step of norm, rotation, write and attend: replayed with other positions, lengths, tables and rows, with
    eager work between, as the eager calls give."""
    from lingbot_world_v2_realtime_amd import KV4Cache, Rotary, norm_rotary_embed
    g = _gen(5)
    hq, hk, d, seqs, pages = 8, 2, 128, 3, 40
    plan, w = Rotary.build(d, DEV), _rand(g, d, mean=1.0, dtype=torch.bfloat16)
    cache, other = _filled(g, pages, hk, d), _filled(_gen(6), pages, hk, d)
    for a, b in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), (other.k, other.k_scale, other.v, other.v_scale)):
        b.copy_(a)
    q, k, v = (_rand(g, seqs, 1, h, d, dtype=torch.bfloat16) for h in (hq, hk, hk))
    pos, lens, table = torch.zeros(seqs, 1, dtype=torch.int32, device=DEV), _dev([1] * seqs), _dev(_table(g, [12] * seqs, pages))

    def step(cache):
        qr, kr = norm_rotary_embed(q, k, pos, plan, w, w)
        cache.write(0, kr[:, 0], v[:, 0], table, lens)
        return cache.attend(0, qr[:, 0], table, lens)

    graph, out = _captured(lambda: step(cache))
    for a, b in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), (other.k, other.k_scale, other.v, other.v_scale)):
        a.copy_(b)
    for n in ([1, 1, 1], [700, 64, 65], [0, 768, 1], [333, 2, 128], [1, 64, 640]):
        for x in (q, k, v):
            x.copy_(_rand(g, *x.shape, dtype=torch.bfloat16))
        lens.copy_(_dev(n))
        pos.copy_(_dev([[max(i - 1, 0)] for i in n]))
        table.copy_(_dev(_table(g, [12] * seqs, pages)))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        want = step(other)
        assert torch.equal(got, want), n
        for a, b in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), (other.k, other.k_scale, other.v, other.v_scale)):
            assert torch.equal(a, b), n


def test_training_in_a_graph():
    """A captured step with its gradients, replayed with other rows and other starts."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    g = _gen(7)
    rows, hq, hk, d = 300, 4, 2, 64
    plan, pos = Rotary.build(d, DEV), torch.arange(rows, device=DEV)
    leaves = [_rand(g, 1, rows, h, d, dtype=torch.bfloat16).requires_grad_() for h in (hq, hk, hk)]
    leaves.append(_rand(g, d, mean=1.0).requires_grad_())
    st, do = _dev([0, 100, 300]), _rand(g, rows, hq, d, dtype=torch.bfloat16)

    def step():
        q, k, v, w = leaves
        qr, kr = norm_rotary_embed(q, k, pos, plan, w, w)
        out = packed_attention(qr[0], kr[0], v[0], st)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    graph, outs = _captured(step)
    for starts in ([0, 100, 300], [0, 0, 300], [20, 280, 290], [0, 299, 300]):
        with torch.no_grad():
            for x in (*leaves, do):
                x.copy_(_rand(g, *x.shape, dtype=x.dtype))
        st.copy_(_dev(starts))
        graph.replay()
        got = [x.clone() for x in outs]
        torch.cuda.synchronize()
        want = step()
        for a, b in zip(got, want):
            assert torch.equal(a, b), starts
        del want


def test_two_streams_at_once():
    """The same calls on two streams beside each other, each with its own tensors, as alone."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    plan, hq, hk, d, lens = Rotary.build(64, DEV), 8, 2, 64, [700, 30, 129]
    st, table, held = _dev(_starts(lens)), _dev([[0, 1, 2, 3], [4, 5, -1, -1], [6, 7, 8, -1]]), _dev([250, 70, 130])

    def work(seed):
        g = _gen(seed)
        x = [_rand(g, 1, sum(lens), h, d, dtype=torch.bfloat16).requires_grad_() for h in (hq, hk, hk)]
        do, one = _rand(g, sum(lens), hq, d, dtype=torch.bfloat16), _rand(g, 3, hq, d, dtype=torch.bfloat16)
        cache = _filled(g, 9, hk, d)
        return x, do, one, cache

    def run(x, do, one, cache):
        qr, kr = norm_rotary_embed(x[0], x[1], 7, plan)
        out = packed_attention(qr[0], kr[0], x[2][0], st)
        return [out.detach(), *torch.autograd.grad(out, x, do), cache.attend(0, one, table, held)]

    ins = [work(s) for s in (1, 2)]
    want = [run(*i) for i in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*ins[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            for a, b in zip(outs, want[i]):
                assert torch.equal(a, b)


def test_gradients_that_are_views():
    """A gradient that is one value expanded, and one whose rows lie apart."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    g = _gen(9)
    q, k, v = (_rand(g, 90, h, 64, dtype=torch.bfloat16).requires_grad_() for h in (4, 2, 2))
    st, plan = _dev([0, 33, 90]), Rotary.build(64, DEV)
    for do in (torch.ones((), dtype=torch.bfloat16, device=DEV).expand(90, 4, 64), _rand(g, 90, 4, 65, dtype=torch.bfloat16)[..., :64],
               _rand(g, 4, 90, 64, dtype=torch.bfloat16).transpose(0, 1), _rand(g, 90, 1, 64, dtype=torch.bfloat16).expand(90, 4, 64)):
        got = torch.autograd.grad(packed_attention(q, k, v, st), (q, k, v), do)
        want = torch.autograd.grad(packed_attention(q, k, v, st), (q, k, v), do.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = torch.autograd.grad(norm_rotary_embed(q[None], None, 3, plan)[0], q, do[None])
        want = torch.autograd.grad(norm_rotary_embed(q[None], None, 3, plan)[0], q, do.contiguous()[None])
        assert torch.equal(got[0], want[0])


# ---------------------------------------------------------------- values that are not finite, where nothing sees them

# heads at which a workgroup takes 64 queries and 32 keys, 64 and 64, 128 and 128, of one sequence of 400
HEADS = [1, 80, 128]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", HEADS)
def test_packed_forms(heads, d, dtype):
    _check_packed(heads, [400], [400], heads, heads, d, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_packed_does_not_see_later_keys(odd, heads, d, dtype):
    """A later key that is not finite leaves the rows before it, and their dq, as they are; a value that is not finite stays in its
    channel of the rows that see it."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g, t, lens, n = _gen(20), DT[dtype], [400, 33], 400
    st = _starts(lens)
    q, k, v, do = (_rand(g, sum(lens), heads, d, dtype=t) for _ in range(4))
    r = causal.packed(q[:, :1], k[:, :1], v[:, :1], st, st, d_out=do[:, :1])
    h = torch.finfo(t).eps / 2
    tol = ((h + _packed_bounds(r, n, d, dtype)) * r["p_v"] + n * 2.0 ** -35)[:, 0]
    for at in (1, 31, 96, 130, 399):
        bad = v.clone()
        bad[at, :, 5] = odd
        out = packed_attention(q, k, bad, _dev(st))
        sees = torch.zeros(sum(lens), dtype=torch.bool, device=DEV)
        sees[at:n] = True
        assert not out[sees][..., 5].isfinite().any(), at
        if odd == odd:
            assert bool((out[sees][..., 5] == odd).all())
        keep = torch.arange(d, device=DEV) != 5
        _within(out[:, 0][:, keep], r["out"][:, 0][:, keep], tol[:, keep], f"value {at}")
        _within(out[~sees][:, 0], r["out"][~sees][:, 0], tol[~sees], f"value {at}")
        kb = k.clone()
        kb[at] = odd
        bad[at] = odd
        leaves = [x.detach().requires_grad_() for x in (q, kb, bad)]
        out = packed_attention(*leaves, _dev(st))
        _within(out.detach()[~sees][:, 0], r["out"][~sees][:, 0], tol[~sees], f"key {at}")
        assert not out.detach()[sees].isfinite().all(-1).any()
        dq, dk, dv = torch.autograd.grad(out, leaves, do)
        steps = E * (n / 16 + 16)
        top = _packed_bounds(r, n, d, dtype).max()
        for x, name, rows in ((dq, "dq", ~sees), (dk, "dk", slice(n, None)), (dv, "dv", slice(n, None))):
            bound = (h + steps) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (top + h * h + E * (d / 16 + 8)) * r[name + "_wide32"]
            _within(x[rows][:, 0], r[name][rows][:, 0], bound[rows][:, 0], f"{name}, key {at}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", HEADS)
def test_packed_gradients_do_not_see_earlier_queries(heads, d, dtype):
    """A query, or its gradient, that is not finite leaves the dk and dv of keys behind it as they are; a gradient that is not
    finite stays in its channel of dv."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g, t, n = _gen(21), DT[dtype], 400
    st = [0, n]
    q, k, v, do = (_rand(g, n, heads, d, dtype=t) for _ in range(4))
    for at in (0, 31, 97, 130, 398):
        keep = torch.ones(n, 1, 1, device=DEV, dtype=t)
        keep[at] = 0   # the gradients without the row are those of a gradient of zeros there
        r = causal.packed(q[:, :1], k[:, :1], v[:, :1], st, st, d_out=(do * keep)[:, :1])
        h, steps, top = torch.finfo(t).eps / 2, E * (n / 16 + 16), _packed_bounds(r, n, d, dtype).max()
        bound = {name: (h + steps) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (top + h * h + E * (d / 16 + 8)) * r[name + "_wide32"]
                 for name in ("dq", "dk", "dv")}
        unseen = torch.arange(n, device=DEV) > at
        others = torch.arange(n, device=DEV) != at
        for what in ("query", "gradient"):
            qb, db = q.clone(), do * keep
            if what == "query":
                qb[at] = float("nan")
            else:
                db[at, :, 5] = float("inf")
            leaves = [x.detach().requires_grad_() for x in (qb, k, v)]
            grads = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(packed_attention(*leaves, _dev(st)), leaves, db)))
            for name, rows in (("dq", others), ("dk", unseen), ("dv", unseen)):
                _within(grads[name][rows][:, 0], r[name][rows][:, 0], bound[name][rows][:, 0], f"{name}, {what} {at}")
            assert not grads["dq"][at].isfinite().any() and not grads["dk"][~unseen].isfinite().any()
            if what == "gradient":
                c = torch.arange(d, device=DEV) != 5
                assert bool((grads["dv"][~unseen][..., 5] == float("inf")).all())
                _within(grads["dv"][:, 0][:, c], r["dv"][:, 0][:, c], bound["dv"][:, 0][:, c], f"dv beside, {at}")


# ---------------------------------------------------------------- sizes


def test_cache_past_two_gib():
    """Pages whose offsets pass 2^31 (and, of all heads' values, 2^32) bytes."""
    g = _gen(30)
    heads, d, pages = 8, 128, 140000   # 4.6 GB each of k and v
    from lingbot_world_v2_realtime_amd import KV4Cache
    big, small = KV4Cache.empty(1, pages, heads, d, DEV), KV4Cache.empty(1, 8, heads, d, DEV)
    lens, new = [200, 70], [200, 40]
    at = _dev([[pages - 1, 65537, 131071, 70000], [3, 139000, -1, -1]])
    near = _dev([[0, 1, 2, 3], [4, 5, -1, -1]])
    st = _dev(_starts(new))
    k, v = (_rand(g, sum(new), heads, d, dtype=torch.bfloat16) for _ in range(2))
    q, one = _rand(g, sum(new), 16, d, dtype=torch.bfloat16), _rand(g, 2, 16, d, dtype=torch.bfloat16)
    tok = _dev([201, 71])
    outs = []
    for cache, table in ((big, at), (small, near)):
        cache.write(0, k, v, table, _dev(lens), st)
        cache.write(0, k[:2], v[:2], table, tok)
        outs.append((*cache.read(0, table, _dev(lens), st, tokens=sum(new)), cache.attend(0, q, table, _dev(lens), st),
                     cache.attend(0, one, table, tok)))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())


def test_packed_and_norm_past_two_to_the_31():
    """Rows behind the 2^31st element, forward and backward."""
    from lingbot_world_v2_realtime_amd import Rotary, norm_rotary_embed, packed_attention
    heads, d, n, seqs = 128, 128, 64, 2100
    rows = n * seqs   # 2.2e9 elements
    g = _gen(31)
    q = torch.empty(rows, heads, d, dtype=torch.bfloat16, device=DEV)
    tail = _rand(g, 2 * n, heads, d, dtype=torch.bfloat16)
    q.view(-1, 2 * n, heads, d).copy_(tail.expand(seqs // 2, *tail.shape))
    k, v = (_rand(g, 2 * n, 1, d, dtype=torch.bfloat16).repeat(seqs // 2, 1, 1) for _ in range(2))
    st, few = _dev([n * i for i in range(seqs + 1)]), _dev([0, n, 2 * n])
    leaves = [x.requires_grad_() for x in (q, k, v)]
    part = [x.detach()[-2 * n:].clone().requires_grad_() for x in (q, k, v)]
    out, want = packed_attention(*leaves, st), packed_attention(*part, few)
    do = _rand(g, 2 * n, heads, d, dtype=torch.bfloat16)
    for x in (out, want):
        assert torch.equal(x.detach()[-2 * n:], want.detach())
    tol = 2.0 ** -7   # (other workgroup sizes: fp32 sums in another order, then rounded: 2 steps)
    for x, y in zip(torch.autograd.grad(out, leaves, do.repeat(seqs // 2, 1, 1)), torch.autograd.grad(want, part, do)):
        big = y.double().abs().amax()
        assert (x[-2 * n:].double() - y.double()).abs().max() <= tol * big
    del out, want, x, y
    plan = Rotary.build(d, DEV)
    with torch.no_grad():
        got = norm_rotary_embed(q[None], None, 0, plan)[0][0, -n:]
        one = norm_rotary_embed(q[None, -n:], None, rows - n, plan)[0][0]
    assert torch.equal(got, one)


def test_norm_rotary_without_eps():
    """eps 0, where lanes of a row's team hold no channel."""
    for d in (2, 40, 80, 129, 250):
        for dtype in DT:
            _check_norm_rotary(d, 1, 5, 3, 2, d, dtype, eps=0.0)


def test_smallest_calls():
    from lingbot_world_v2_realtime_amd import KV4Cache, packed_attention
    g = _gen(40)
    q = _rand(g, 1, 1, 64, dtype=torch.bfloat16)
    assert torch.equal(packed_attention(q, q, q, _dev([0, 1])), q)
    cache = KV4Cache.empty(1, 1, 1, 64, DEV)
    x = causal.values(*causal.encode(q)).bfloat16()
    cache.write(0, q, q, _dev([[0]]), _dev([1]))
    assert torch.equal(cache.attend(0, q, _dev([[0]]), _dev([1])), x)
    assert not cache.attend(0, q, _dev([[0]]), _dev([0])).any()


@pytest.mark.parametrize("width", [3, 60])
@pytest.mark.parametrize("seqs", [40, 200])
def test_cache_with_falling_starts(seqs, width):
    """Starts that fall have no particular answer; the calls end, stay inside their tensors, and leave what the table does not name."""
    g = _gen(41)
    rows, heads, d = 8, 2, 64
    cache = _filled(g, 3 * seqs, heads, d)
    before = [x.clone() for x in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
    q, k, v = (_rand(g, rows, h, d, dtype=torch.bfloat16) for h in (4, heads, heads))
    table, lens = _dev([[i, -1, 2 * seqs + i] + [-1] * (width - 3) for i in range(seqs)]), _dev([150] * seqs)
    for starts in ([0, rows] * (seqs // 2) + [0], [rows] * seqs + [0], [0] + [2 ** 31 - 1, -5] * (seqs // 2)):
        args = (table, lens, _dev(starts))
        cache.attend(0, q, *args)
        cache.read(0, *args, tokens=rows)
        cache.write(0, k, v, *args)
    torch.cuda.synchronize()
    for x, y in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), before):
        assert torch.equal(x[:, seqs:2 * seqs], y[:, seqs:2 * seqs])


@pytest.mark.parametrize("d,dtype", [(64, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 300])
def test_cache_attend_shares_of_many_sequences(seqs, d, dtype):
    """Keys shared evenly over waves, of more sequences than a wave has lanes (a wide table says that they may be long): single
    tokens, and a few or none of each; lengths of 0, some that end a page."""
    lens = [(67 * i) % 190 for i in range(seqs)]
    lens[seqs // 2] = 1500
    _check_cache_attend(seqs, [1] * seqs, lens, 4, 2, d, dtype, width=60, starts=False)
    _check_cache_attend(seqs + 1, [(i * 7) % 4 for i in range(seqs)], lens, 6, 1, d, dtype, width=100)


def test_cache_attend_whole_tiles():
    """Each tile of rows by a wave of its own: many sequences under a narrow table, several tokens, many heads."""
    lens = [(67 * i) % 250 for i in range(150)]
    for dtype in DT:
        if dtype != "fp32":
            _check_cache_attend(50, [1] * 150, lens, 4, 2, 128, dtype, starts=False)
            _check_cache_attend(51, [(i * 7) % 8 for i in range(150)], lens, 20, 1, 64, dtype, tail=3)


@pytest.mark.parametrize("hq,hk", [(96, 12), (45, 45), (24, 24), (48, 24), (36, 36)])
@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
def test_packed_forms_of_several_sequences(hq, hk, d, dtype):
    """Each size of a workgroup's tile over sequences of different lengths, heads that share XCDs in every way."""
    _check_packed(hq + hk, [300, 0, 77, 129, 5, 640], [300, 12, 140, 100, 5, 640], hq, hk, d, dtype, tail=2)


@pytest.mark.parametrize("seqs", [61, 62, 63])
def test_packed_as_many_sequences_as_a_wave_looks_at(seqs):
    lens = [(53 * i) % 170 for i in range(seqs)]
    _check_packed(seqs, lens, [max(0, n + i % 5 - 2) for i, n in enumerate(lens)], 2, 1, 64, head=3, tail=5)


def test_packed_is_the_same_every_time():
    """No sum has an order of its own: a training step's bits, over and over, beside other work."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g = _gen(60)
    lens = [900, 33, 400, 128]
    q, k, v = (_rand(g, sum(lens), h, 128, dtype=torch.bfloat16).requires_grad_() for h in (12, 4, 4))
    do, st = _rand(g, sum(lens), 12, 128, dtype=torch.bfloat16), _dev(_starts(lens))
    other, noise = torch.cuda.Stream(), torch.randn(2048, 2048, device=DEV)
    want = None
    for _ in range(6):
        with torch.cuda.stream(other):
            noise = noise @ noise * 1e-2
        out = packed_attention(q, k, v, st)
        got = (out.detach(), *torch.autograd.grad(out, (q, k, v), do))
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
