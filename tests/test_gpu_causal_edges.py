"""Causal self-attention at the edges of what its calls allow: starts that have no meaning, which must leave every tensor's
surroundings alone, lengths past a table's width, infinities that leave a row no softmax, rows and tables that lie anywhere, and as many
sequences and heads as there may be. Bounds as in test_gpu_causal.py.
"""
import pytest
import torch

from oracle import causal
from test_gpu_causal import DEV, DT, E, _dev, _filled, _gen, _packed_bounds, _rand, _starts, _table, _together, _within

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- starts that fall


def _falling(seqs, rows):
    """Starts of `seqs` sequences that rise and fall: searches among them end at sequences that begin behind what is searched."""
    return {"up and down": ([0, rows] * (seqs + 1))[:seqs + 1], "saw": [97 * i % rows for i in range(seqs + 1)],
            "one fall": [rows] * seqs + [0], "out of range": ([0] + [2 ** 31 - 1, -5] * seqs)[:seqs + 1]}


class _Guarded:
    """Tensors in the middle of larger ones, whose ends hold one value and have to go on doing so."""

    def __init__(self, margin):
        self.margin, self.all = margin, []

    def make(self, x, value):
        flat = torch.full((x.numel() + 2 * self.margin,), value, dtype=x.dtype, device=DEV)
        inner = flat[self.margin:self.margin + x.numel()].view(x.shape)
        inner.copy_(x)
        self.all.append((flat, x.numel(), value))
        return inner

    def check(self):
        for flat, n, value in self.all:
            for end in (flat[:self.margin], flat[self.margin + n:]):
                assert bool(end.isnan().all() if value != value else (end == value).all())


@pytest.mark.parametrize("seqs", [63, 64, 65, 200])
@pytest.mark.parametrize("heads", [1, 40])
def test_packed_with_falling_starts(lib, seqs, heads):
    """No particular answer, but nothing outside is read (NaN lies there, and the outputs are finite) or written."""
    rows, d, g = 300, 64, _gen(seqs)
    stream = torch.cuda.current_stream().cuda_stream
    nan = float("nan")
    for name, st in _falling(seqs, rows).items():
        for starts, k_starts in ((st, st), (_starts([0] * (seqs - 1) + [rows]), st), (st, _starts([0] * (seqs - 1) + [rows]))):
            box = _Guarded(8192 * heads)
            q, k, v, do = (box.make(_rand(g, rows, heads, d, dtype=torch.bfloat16), nan) for _ in range(4))
            zero = torch.zeros_like(q)
            out, rest, dq, dk, dv = (box.make(zero, 7.0) for _ in range(5))
            lse, ws = (box.make(torch.zeros(heads, rows, device=DEV), 7.0) for _ in range(2))
            a, b = _dev(starts), _dev(k_starts)
            strides = [heads * d, d]
            assert lib.lbw_packed_attn_bwd_workspace_bytes(rows, rows, heads, heads) <= 4 * ws.numel()
            assert lib.lbw_packed_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), 0, seqs, rows, rows, heads, heads, d, *strides * 3, a.data_ptr(),
                                           b.data_ptr(), 1, 0.125, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), stream) == 0
            assert lib.lbw_packed_attn_bwd(do.data_ptr(), out.data_ptr(), rest.data_ptr(), lse.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), 0,
                                           seqs, rows, rows, heads, heads, d, *strides * 4, a.data_ptr(), b.data_ptr(), 1, 0.125, dq.data_ptr(),
                                           dk.data_ptr(), dv.data_ptr(), ws.data_ptr(), stream) == 0
            torch.cuda.synchronize()
            box.check()
            assert all(bool(x.isfinite().all()) for x in (out, dq, dk, dv)), name


@pytest.mark.parametrize("width", [2, 60])
@pytest.mark.parametrize("rows", [8, 300])
@pytest.mark.parametrize("seqs", [40, 64, 200])
def test_cache_with_falling_starts_stays_inside(lib, seqs, rows, width):
    """The cache's calls, by a wave a tile (narrow tables) and shared (wide ones): NaN around every input and in front of the
    workspace, whose own words claim that a tile has two segments; nothing outside an output changes."""
    heads, hq, d, g = 2, 4, 64, _gen(rows + seqs)
    stream = torch.cuda.current_stream().cuda_stream
    nan = float("nan")
    table, lens = _dev([[i, seqs + i] + [-1] * (width - 2) for i in range(seqs)]), _dev([128] * seqs)
    for name, st in _falling(seqs, rows).items():
        box = _Guarded(1 << 16)
        q, k, v = (box.make(_rand(g, rows, h, d, dtype=torch.bfloat16), nan) for h in (hq, heads, heads))
        out, rk, rv = (box.make(torch.zeros(rows, h, d, dtype=torch.bfloat16, device=DEV), 7.0) for h in (hq, heads, heads))
        cache, starts = _filled(g, 2 * seqs, heads, d), _dev(st)
        parts = [box.make(x.view(-1), 7).view(x.shape) for x in (cache.k, cache.k_scale, cache.v, cache.v_scale)]
        call = (starts.data_ptr(), lens.data_ptr(), table.data_ptr(), width, width, 2 * seqs, *(x.data_ptr() for x in parts))
        bytes_ = lib.lbw_kv4_attn_workspace_bytes(seqs, rows, hq, heads, d, width, 0)
        assert (bytes_ > 0) == (16 * width > rows + 40)
        ws = torch.full((bytes_ // 4 + (2 << 16),), nan, device=DEV)
        inner = ws[1 << 16:(1 << 16) + bytes_ // 4]
        inner.fill_(1.0)
        places = rows // 8 + seqs if bytes_ else 0   # (two words for each tile of 8 tokens lie at the end: its first segment and its last)
        inner[inner.numel() - 2 * places:].view(torch.int32).copy_(torch.arange(2 * places, device=DEV) % 2)
        assert lib.lbw_kv4_attn(q.data_ptr(), 0, seqs, rows, hq, heads, d, hq * d, d, *call, 0.125, out.data_ptr(), inner.data_ptr(), stream) == 0
        assert lib.lbw_kv4_read(seqs, rows, heads, d, *call, rk.data_ptr(), rv.data_ptr(), stream) == 0
        assert lib.lbw_kv4_write(k.data_ptr(), v.data_ptr(), 0, seqs, rows, heads, d, *[heads * d, d] * 2, *call, stream) == 0
        torch.cuda.synchronize()
        box.check()
        assert bool(ws[:1 << 16].isnan().all() and ws[(1 << 16) + bytes_ // 4:].isnan().all())
        assert all(bool(x.isfinite().all()) for x in (out, rk, rv)), name


# ---------------------------------------------------------------- lengths past the table


@pytest.mark.parametrize("counts,lens,width,hq,hk", [
    ([5], [130], 2, 4, 2), ([10], [70], 1, 4, 1), ([3, 70, 5], [129, 150, 64], 2, 8, 2),   # a wave a tile
    ([5, 9], [258, 300], 4, 4, 2), ([2, 1, 6], [700, 257, 255], 4, 40, 1), ([20], [3010], 47, 2, 2),   # shared
    ([1, 30], [100, 2000], 1, 6, 3), ([7, 0, 3], [2 ** 31 - 1, 500, 66], 1, 2, 1)])
@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
def test_cache_attend_of_lengths_past_the_table(counts, lens, width, hq, hk, d, dtype):
    """A row's place is that of write and read, whatever the table holds: rows inside it see the tokens up to their own, rows
    past it all that there are."""
    short = [min(n, 64 * width) for n in lens]
    g = _gen(sum(counts))
    st, t = _starts(counts, 2), DT[dtype]
    pages = sum(-(-n // 64) for n in short) + 2
    cache, table = _filled(g, pages, hk, d), _table(g, [-(-n // 64) for n in short], pages, width)
    q = _rand(g, st[-1] + 3, hq, d, dtype=t)
    out = cache.attend(0, q, _dev(table), _dev(lens), _dev(st))
    assert torch.equal(out, cache.attend(0, q, _dev(table), _dev(lens), _dev(st)))
    r = causal.cache_attend(q, *causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0]), st, lens, table)
    h = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -16
    _within(out, r["out"], (h + _packed_bounds(r, max(short), d, dtype)) * r["p_v"], f"{counts} of {lens}, {width} pages")
    _together(out, r["out"], r["p2_v2"], f"{counts} of {lens}")


def test_cache_rows_past_the_table_see_what_was_written():
    """Written, read back and attended: a row whose own token lies inside the table answers as it does with a wider table."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    g = _gen(71)
    cache, st = KV4Cache.empty(1, 3, 2, 128, DEV), _dev([0, 60])
    k, v = (_rand(g, 130, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    q, wide, narrow = _rand(g, 60, 4, 128, dtype=torch.bfloat16), _dev([[2, 0, 1]]), _dev([[2, 0]])
    cache.write(0, k, v, wide, _dev([130]), _dev([0, 130]))
    a, b = (cache.attend(0, q, t, _dev([130]), st) for t in (wide, narrow))
    assert torch.equal(a[:58], b[:58]) and not torch.equal(a[58:], b[58:])
    for row, n in ((0, 71), (57, 128), (59, 128)):
        assert torch.equal(b[row], cache.attend(0, q[row:row + 1], narrow, _dev([n]))[0])


# ---------------------------------------------------------------- scores that are all minus infinity


def _held_together(x, value, bound, what):
    """NaN where the definition has it, and within its bound elsewhere."""
    assert torch.equal(x.isnan(), value.isnan()), what
    keep = ~value.isnan()
    _within(x[keep], value[keep], bound.expand_as(value)[keep], what)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [1, 80, 128])   # (the forms of a workgroup's tile)
@pytest.mark.parametrize("causal_", [True, False])
def test_packed_scores_of_minus_infinity(causal_, heads, d, dtype):
    """A query whose infinity makes every score that it sees minus infinity has no softmax: its row is NaN, as the definition has
    it, not the zeros of a row that sees nothing; so is its gradient, and those of the keys that it sees."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g, t, lens, n = _gen(80), DT[dtype], [400, 33], 400
    st = _starts(lens)
    q, k, v, do = (_rand(g, sum(lens), heads, d, dtype=t) for _ in range(4))
    k[..., 0] = k[..., 0].abs() + 0.125
    rows = torch.arange(sum(lens), device=DEV)
    for at in (0, 31, 130, 399):
        bad, keep = q.clone(), (rows != at)[:, None, None]
        bad[at, :, 0] = -float("inf")
        leaves = [x.detach().requires_grad_() for x in (bad, k, v)]
        out = packed_attention(*leaves, _dev(st), causal=causal_)
        with torch.no_grad():
            assert packed_attention(*leaves, _dev(st), causal=causal_)[at].isnan().all()
        # (what the other rows have is what they have where this one's gradient is zero)
        r = causal.packed(q[:, :1], k[:, :1], v[:, :1], st, st, causal=causal_, d_out=(do * keep)[:, :1])
        h, rel = torch.finfo(t).eps / 2, _packed_bounds(r, n, d, dtype)
        nan = torch.full((), float("nan"), dtype=torch.float64, device=DEV)
        _held_together(out.detach()[:, :1], r["out"].where(keep, nan), (h + rel) * r["p_v"] + n * 2.0 ** -35, f"row {at}")
        steps, top = E * (n / 16 + 16), rel.max()
        unseen = ((rows > at) if causal_ else (rows >= n))[:, None, None]
        for x, name in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv")):
            bound = (h + steps) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (top + h * h + E * (d / 16 + 8)) * r[name + "_wide32"]
            _held_together(x[:, :1], r[name].where(keep if name == "dq" else unseen, nan), bound, f"{name}, row {at}")


def test_packed_key_of_minus_infinity():
    """The same from a key's infinity: the row that sees it alone is NaN, those behind it give it no weight."""
    from lingbot_world_v2_realtime_amd import packed_attention
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        g = _gen(81)
        q, k, v = (_rand(g, 70, 2, d, dtype=dtype) for _ in range(3))
        q[..., 0] = q[..., 0].abs() + 0.125
        k[0, :, 0] = -float("inf")
        out = packed_attention(q, k, v, _dev([0, 70]))
        r = causal.packed(q, k, v, [0, 70], [0, 70])
        assert out[0].isnan().all() and out[1:].isfinite().all()
        h = torch.finfo(dtype).eps / 2
        k[0, :, 0] = 0
        rel = _packed_bounds(causal.packed(q, k, v, [0, 70], [0, 70]), 70, d, dtype)
        _held_together(out, r["out"], (h + rel) * v.double().abs().amax() + 70 * 2.0 ** -35, "out")


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("width,lens,counts", [(6, [130, 290, 40], [1, 1, 1]), (60, [130, 3000, 64], [1, 1, 1]), (60, [130, 3000, 40], [5, 2, 3]), (6, [130, 290, 40], [50, 20, 9])])
def test_cache_scores_of_minus_infinity(width, lens, counts, d, dtype):
    """The cache's attention likewise, by a wave and shared: a query's infinity against positive keys. Rows that see nothing, and rows
    whose pages are all missing, stay zero."""
    g, t = _gen(83), DT[dtype]
    hq, hk, st = 6, 2, _starts(counts)
    cache = _filled(g, 60, hk, d)
    cache.k[..., 0] = cache.k[..., 0] & 0xF7 | 1   # channel 0 (a token's first code): 0.5 or more
    table = _table(g, [-(-n // 64) for n in lens], 60, width)
    table[2][0] = -1                               # the third sequence's only page
    q = _rand(g, st[-1], hq, d, dtype=t)
    one = counts == [1, 1, 1]
    args = (_dev(table), _dev(lens), None if one else _dev(st))
    want = cache.attend(0, q, *args)
    kv = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    assert bool((kv[0][..., 0] > 0).all())
    for at in (0, st[1], st[2], st[3] - 1):
        bad = q.clone()
        bad[at, 1, 0] = -float("inf")
        got = cache.attend(0, bad, *args)
        keep = torch.ones(st[-1], hq, 1, dtype=torch.bool, device=DEV)
        keep[at, 1] = at >= st[2]   # (the third's rows see no page that there is)
        assert torch.equal(got.isnan(), ~keep.expand_as(got)), at
        assert torch.equal(got.where(keep, torch.zeros_like(got)), want.where(keep, torch.zeros_like(got))), at
        if at >= st[2]:
            assert not got[at].any()


def test_cache_scores_of_minus_infinity_in_a_part(lib):
    """Scores that overflow to minus infinity over some of a row's pages and not over others: those weigh nothing."""
    g = _gen(84)
    cache = _filled(g, 60, 1, 64)
    cache.k[..., 0] = cache.k[..., 0] & 0xF0 | 0xC     # channel 0: -2
    cache.k_scale[..., 0] = 127
    table = _dev([list(range(60))])
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device=DEV)
    q[0, 0, 0] = 2.0 ** 127
    want = cache.attend(0, q, table, _dev([3840]), sm_scale=1.0)
    assert want.isnan().all()                            # (every score is -2^128)
    few = [7, 1000, 3839]
    for t in few:
        cache.k[0, t // 64, 0, t % 64, 0] &= 0xF0        # 0
    got = cache.attend(0, q, table, _dev([3840]), sm_scale=1.0)
    _, v = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    mean = sum(v[t // 64, 0, t % 64] for t in few) / len(few)
    _within(got[0, 0], mean, 2.0 ** -22 * mean.abs(), "three keys alike")


def _grads_of_a_key_of_minus_infinity(heads, d, dtype, causal_, names):
    """One key whose infinity makes its scores minus infinity, for every row that sees it: its weights are zero, and the other
    rows' and keys' gradients those without it. Checks the first head's."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g, t, n = _gen(82), DT[dtype], 400
    q, k, v, do = (_rand(g, n, heads, d, dtype=t) for _ in range(4))
    q[..., 0] = q[..., 0].abs() + 0.125
    for at in (1, 31, 96, 130, 399):
        bad, see, zero = k.clone(), causal.visible(n, n, causal_, DEV), k.clone()
        bad[at, :, 0], zero[at, :, 0], see[:, at] = -float("inf"), 0, False
        leaves = [x.detach().requires_grad_() for x in (q, bad, v)]
        out = packed_attention(*leaves, _dev([0, n]), causal=causal_)
        r = causal.attend(q[:, 0], zero[:, 0], v[:, 0], see, d ** -0.5, do[:, 0])
        h, rel = torch.finfo(t).eps / 2, _packed_bounds(r, n, d, dtype)
        _held_together(out.detach()[:, 0], r["out"], (h + rel) * r["p_v"] + n * 2.0 ** -35, f"out, key {at}")
        # zero times its infinity is no number: in its channel, for every row that sees it
        r["dq"][torch.arange(n, device=DEV) >= (at if causal_ else 0), 0] = float("nan")
        steps, top = E * (n / 16 + 16), rel.max()
        for x, name in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv")):
            if name in names:
                bound = (h + steps) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (top + h * h + E * (d / 16 + 8)) * r[name + "_wide32"]
                _held_together(x[:, 0], r[name], bound, f"{name}, key {at}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [1, 80, 128])
@pytest.mark.parametrize("causal_", [True, False])
def test_packed_gradients_of_a_key_beside_rows_behind_the_last(causal_, heads, d, dtype):
    """Rows behind the last query, which fill its tile, are no queries: such a key's dk and dv are zero, not NaN."""
    _grads_of_a_key_of_minus_infinity(heads, d, dtype, causal_, ("dk", "dv"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [1, 80, 128])
@pytest.mark.parametrize("causal_", [True, False])
def test_packed_gradient_of_rows_that_see_a_key_of_minus_infinity(causal_, heads, d, dtype):
    """dq is NaN in the infinity's channel for the rows that see it, in a tile that is partly seen or wholly, and there alone."""
    _grads_of_a_key_of_minus_infinity(heads, d, dtype, causal_, ("dq",))


# ---------------------------------------------------------------- rows and tables that lie anywhere


@pytest.mark.parametrize("d,dtype", [(64, "fp16"), (128, "bf16")])
@pytest.mark.parametrize("counts", [[1, 1, 1], [70, 5, 33]])
def test_cache_calls_of_views(counts, d, dtype):
    """Parts of one projection, rows that the kernels do not load from (copied), one row for all heads, a table that is a part of a
    wider one, and one row of it for every sequence: as their contiguous copies."""
    from lingbot_world_v2_realtime_amd import KV4Cache
    g, t, hq, hk, st = _gen(90), DT[dtype], 4, 2, _starts(counts)
    rows, starts = st[-1], None if counts == [1, 1, 1] else _dev(st)

    def fused(h):
        return _rand(g, rows, h + 5, d, dtype=t)[:, 3:3 + h]

    def odd(h):
        return _rand(g, rows, h, d + 3, dtype=t)[..., 1:d + 1]

    def turned(h):
        return _rand(g, h, rows, d, dtype=t).transpose(0, 1)

    def spread(h):
        return _rand(g, rows, 1, d, dtype=t).expand(rows, h, d)

    wide = _dev(_table(g, [3, 3, 3], 12, 9))
    for make in (fused, odd, turned, spread):
        for table, lens in ((wide[:, :3], _dev([130, 190, 64])), (wide[:1, :3].expand(3, 3), _dev([130] * 3))):
            k, v, q = make(hk), make(hk), make(hq)
            cache, other = (KV4Cache(*(x.clone() for x in (c.k, c.k_scale, c.v, c.v_scale))) for c in [_filled(_gen(91), 12, hk, d)] * 2)
            args, plain = (table, lens, starts), (table.contiguous(), lens, starts)
            if table.stride(0):   # (a page may be in the table once for the tokens of a write)
                cache.write(0, k, v, *args)
                other.write(0, k.contiguous(), v.contiguous(), *plain)
                assert all(torch.equal(a, b) for a, b in zip((cache.k, cache.k_scale, cache.v, cache.v_scale), (other.k, other.k_scale, other.v, other.v_scale)))
            assert torch.equal(cache.attend(0, q, *args), other.attend(0, q.contiguous(), *plain))
            tokens = None if starts is None else rows
            assert all(torch.equal(a, b) for a, b in zip(cache.read(0, *args, tokens=tokens), other.read(0, *plain, tokens=tokens)))


def test_as_many_sequences_and_heads_as_there_may_be(lib):
    """65535 sequences, most of them empty; 4096 heads."""
    from lingbot_world_v2_realtime_amd import packed_attention
    g, seqs = _gen(92), 65535
    lens = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    for s, n in ((0, 3), (63, 70), (64, 1), (40000, 130), (65534, 65)):
        lens[s] = n
    st = torch.cat((torch.zeros(1, device=DEV), lens.cumsum(0))).int()
    few = _dev([0, 3, 73, 74, 204, 269])
    leaves = [_rand(g, 269, h, 64, dtype=torch.bfloat16).requires_grad_() for h in (2, 1, 1)]
    do = _rand(g, 269, 2, 64, dtype=torch.bfloat16)
    out, want = packed_attention(*leaves, st), packed_attention(*leaves, few)
    r = causal.packed(*(x.detach() for x in leaves), few.tolist(), few.tolist(), d_out=do)
    h = 2.0 ** -8
    rel = _packed_bounds(r, 130, 64, "bf16")
    for x in (out, want):
        _within(x.detach(), r["out"], (h + rel) * r["p_v"] + 130 * 2.0 ** -35, "out")
    for x, name in zip(torch.autograd.grad(out, leaves, do), ("dq", "dk", "dv")):
        bound = (h + E * (130 / 8 + 16)) * r[name + "_abs"] + (h + h * h) * r[name + "_wide16"] + (rel.max() + h * h + 12 * E) * r[name + "_wide32"]
        _within(x, r[name], bound, name)
    cache = _filled(g, 8, 1, 64)
    table = torch.full((seqs, 3), -1, dtype=torch.int32, device=DEV)
    held = torch.zeros(seqs, dtype=torch.int32, device=DEV)
    table[40000], table[65534, :2] = _dev([3, 5, 1]), _dev([0, 7])
    held[40000], held[65534], held[5] = 150, 66, 9
    q = _rand(g, 269, 2, 64, dtype=torch.bfloat16)
    kv = causal.unpack_pages(cache.k[0], cache.k_scale[0], cache.v[0], cache.v_scale[0])
    got = cache.attend(0, q, table, held, st)
    r = causal.cache_attend(q, *kv, [74, 204, 269], [150, 66], [[3, 5, 1], [0, 7]])
    _within(got, r["out"], (h + _packed_bounds(r, 150, 64, "bf16")) * r["p_v"], "attend")
    rows = _rand(g, seqs, 2, 64, dtype=torch.bfloat16)
    one = cache.attend(0, rows, table, held)
    seen = torch.zeros(seqs, dtype=torch.bool, device=DEV)
    seen[40000] = seen[65534] = True
    assert not one[~seen].any() and bool(one[seen].any(-1).all())
    r = causal.cache_attend(rows[seen], *kv, [0, 1, 2], [150, 66], [[3, 5, 1], [0, 7]])
    _within(one[seen], r["out"], (h + _packed_bounds(r, 150, 64, "bf16")) * r["p_v"], "attend, one token each")
    q, k, v = (_rand(g, 5, n, 64, dtype=torch.bfloat16) for n in (4096, 4096, 4096))
    out = packed_attention(q, k, v, _dev([0, 5]))
    one = packed_attention(q[:, -1:], k[:, -1:], v[:, -1:], _dev([0, 5]))
    assert torch.equal(out[:, -1:], one)
    cache = _filled(g, 2, 4096, 64)
    a, b = (cache.attend(0, x, _dev([[1]]), _dev([5]), _dev([0, 5])) for x in (q, q))
    small = type(cache)(*(x[:, :, -1:].contiguous() for x in (cache.k, cache.k_scale, cache.v, cache.v_scale)))
    assert torch.equal(a, b) and torch.equal(a[:, -1:], small.attend(0, q[:, -1:], _dev([[1]]), _dev([5]), _dev([0, 5])))
