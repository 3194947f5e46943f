"""osmos_rope and osmos_rope_append against their formulas in float64, with the errors that the arithmetic may make: the angle's
fraction is exact to 2^-50 of a turn, a sine or cosine off by at most 2^-22 (the angle's rounding to float 0.8 x 2^-24, the series'
few roundings, the factor's), a product and a sum by 2^-24 each: 2^-21 of |a| + |b| in all; a norm's sum of dim squares (13 roundings
in a row), square root, quotient and two products by 2^-20 of the value; then the output's rounding."""
import ctypes
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from libosmos_amd import attn, capi, rows  # noqa: E402

F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _make(shape, kind, seed, rms=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * rms).to(kind)


def _want(table, x, pos, pairs, weight, eps, offset):
    """(the turned heads in float64, the error allowed before the output's rounding)"""
    rot, d, x = table.rot, x.shape[2], x.double()
    rel = 2.0 ** -21
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(2, keepdim=True) + eps) * (weight.double() + offset)
        rel += 2.0 ** -20
    t = (pos.double()[:, None] * table.turns) % 1.0 * (2 * math.pi)
    c, s = (f(t)[:, None] * table.scale for f in (torch.cos, torch.sin))
    y, e = x.clone(), x.abs() * (2.0 ** -20 if weight is not None else 0.0)
    at = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., at[0]], x[..., at[1]]
    y[..., at[0]], y[..., at[1]] = a * c - b * s, b * c + a * s
    for i in at:
        e[..., i] = (a.abs() + b.abs()) * max(1.0, table.scale) * rel
    return y, e


def _near(got, want, e, what):
    e = e + (want.abs() + e) * HALF[got.dtype] + (2.0 ** -25 if got.dtype == F16 else 0.0)
    off = (got.double() - want).abs()
    assert (off <= e).all(), "%s: off by %.3g where %.3g is allowed" % (what, float(off[off > e].max()), float(e[off > e].min()))


SCALINGS = [None, dict(kind="linear", factor=4.0), dict(kind="ntk", factor=8.0), dict(kind="yarn", factor=16.0, context=4096, fast=32.0, slow=1.0),
            dict(kind="bands", factor=8.0, context=8192, low=1.0, high=4.0)]


@pytest.mark.parametrize("dim,rot", [(8, 2), (8, 8), (16, 6), (64, 64), (80, 20), (80, 80), (96, 24), (128, 128), (128, 64), (192, 50), (256, 256), (248, 62)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("kind,out_kind", [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16), (BF16, F32)], ids=str)
def test_rows(dim, rot, pairs, kind, out_kind):
    print(dim, rot, pairs, kind, out_kind, flush=True)
    n, heads, kv = 5, 7, 3
    table = rows.RopeTable(rot, scaling=SCALINGS[(dim + rot) % 5] if rot > 2 else None)
    qk = _make((n, heads + kv + 2, dim), kind, dim + rot)
    q, k = qk[:, :heads], qk[:, heads:heads + kv]
    pos = _ints([0, 1, 131071, -5, 2 ** 30 + 77])
    out, k_out = torch.full((n, heads, dim), 7.0, dtype=out_kind, device="cuda"), torch.full((n, kv, dim), 7.0, dtype=out_kind, device="cuda")
    for qw, kw, offset in ((None, None, 0.0), (_make((dim,), F32, 1), _make((dim,), F32, 2), 1.0), (None, _make((dim,), F32, 3), 0.0)):
        rows.Rope(table, pos, q, out, k, k_out, pairs=pairs, q_weight=qw, k_weight=kw, eps=1e-5, offset=offset).run()
        for got, x, w, what in ((out, q, qw, "q"), (k_out, k, kw, "k")):
            _near(got, *_want(table, x, pos, pairs, w, 1e-5, offset), what)
    if kind == out_kind:  # in place
        want = (out.clone(), k_out.clone())
        rows.Rope(table, pos, q, q, k, k, pairs=pairs, k_weight=kw, eps=1e-5).run()
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.parametrize("n,heads,kv", [(1, 1, 0), (1, 33, 1), (200, 5, 0), (4099, 2, 1), (9000, 1, 0)])
def test_many_rows(n, heads, kv):
    print(n, heads, kv, flush=True)
    table, dim = rows.RopeTable(64), 64
    q = _make((n, heads, dim), F32, 1)
    k = _make((n, kv, dim), F32, 2) if kv else None
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 37 - 100
    out, k_out = torch.empty_like(q), torch.empty_like(k) if kv else None
    rows.Rope(table, pos, q, out, k, k_out).run()
    _near(out, *_want(table, q, pos, False, None, 0.0, 0.0), "q")
    if kv:
        _near(k_out, *_want(table, k, pos, False, None, 0.0, 0.0), "k")


@pytest.mark.parametrize("pairs", [False, True])
def test_what_does_not_turn(pairs):
    """values past the rotary ones, infinities and NaN among them, keep their bits; an infinity in a pair stays in it"""
    table = rows.RopeTable(32)
    q = _make((3, 2, 64), F32, 1)
    q[0, 0, 40], q[1, 1, 63], q[2, 0, 33] = math.inf, math.nan, -0.0
    q[2, 1, 3] = math.inf
    out = torch.empty_like(q)
    rows.Rope(table, _ints([3, 4, 5]), q, out, pairs=pairs).run()
    assert torch.equal(out[..., 32:].contiguous().view(torch.int32), q[..., 32:].contiguous().view(torch.int32))
    bad = ~torch.isfinite(out[..., :32])
    assert bad.sum() == 2 and bad[2, 1, 3] and bad[2, 1, 2 if pairs else 19]


def test_heads_apart():
    """(heads, rows, dim) buffers, and rows out of wider ones"""
    table, pos = rows.RopeTable(48), _ints([9, 8, 7, 6])
    q = _make((5, 4, 64), BF16, 1).permute(1, 0, 2)
    out = torch.full((4, 6, 72), 3.0, dtype=BF16, device="cuda")
    rows.Rope(table, pos, q, out[:, :5, :64]).run()
    _near(out[:, :5, :64], *_want(table, q, pos, False, None, 0.0, 0.0), "q")
    assert (out[:, 5] == 3).all() and (out[:, :, 64:] == 3).all()


class Paged:
    """a step of sequences over a cache with its pages dealt out in reverse"""

    def __init__(self, kind, heads, dim, page, lens, counts, layers=2, seq=None, live=None, extra=0, max_len=None):
        need = [-(-m // page) for m in lens]
        pages, width = sum(need) + 2, max(need) + 1
        scale = 0.01 + 0.02 * torch.rand((layers, 2, heads), device="cuda") if kind == F8 else None
        self.cache = attn.KvCache.empty(kind, layers, pages, heads, page, dim, scale)
        self.cache.data.view(torch.uint8).fill_(0x3A)
        ids = list(range(pages))[::-1]
        self.rows = [[ids.pop() for _ in range(k)] for k in need]
        self.table = _ints([r + [-1] * (width - len(r)) for r in self.rows])
        self.lens, self.counts = lens, counts
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        self.n = starts[-1] + extra
        self.step = attn.KvStep(_ints(starts), _ints(lens), self.table, n_tok=self.n, max_tok=max(max(counts), 1), max_len=max_len or max(lens),
                                seq=None if seq is None else _ints(seq), live=None if live is None else _ints(live))


@pytest.mark.parametrize("kind,cache", [(F32, F16), (F32, F8), (F16, F16), (BF16, BF16), (BF16, F8), (F16, BF16)], ids=str)
@pytest.mark.parametrize("heads,kv,dim,rot,pairs", [(8, 2, 64, 64, False), (3, 3, 80, 20, True), (4, 1, 256, 64, False), (6, 2, 192, 192, True),
                                                     (5, 5, 48, 22, False)])
def test_append(kind, cache, heads, kv, dim, rot, pairs):
    """the cache's bits are those of osmos_rope into float rows and osmos_kv_append of these, q's those of osmos_rope"""
    print(kind, cache, heads, kv, dim, rot, pairs, flush=True)
    lens, counts = [40, 1, 17, 300], [7, 1, 0, 33]
    p = Paged(cache, kv, dim, 16, lens, counts)
    n, table = p.n, rows.RopeTable(rot)
    qkv = _make((n, heads + 2 * kv, dim), kind, dim, 2.0)
    q, k, v = qkv.split([heads, kv, kv], 1)
    qw, kw = (_make((dim,), F32, 5), _make((dim,), F32, 6)) if heads % 2 else (None, None)
    args = dict(pairs=pairs, q_weight=qw, k_weight=kw, eps=1e-5, offset=0.25)
    pos = _ints([m - c + i for m, c in zip(lens, counts) for i in range(c)])
    out, want = torch.empty((n, heads, dim), dtype=kind, device="cuda"), torch.empty((n, heads, dim), dtype=kind, device="cuda")
    k32 = torch.empty((n, kv, dim), device="cuda")
    rows.Rope(table, pos, q, want, **args).run()
    rows.Rope(table, pos, k, k32, **dict(args, q_weight=kw)).run()
    before = p.cache.data.clone()
    attn.Append(p.cache, 1, p.step, k32, v.float().contiguous()).run()
    kept = p.cache.data.clone()
    assert not torch.equal(kept.view(torch.uint8), before.view(torch.uint8))
    p.cache.data.copy_(before)
    rows.RopeAppend(table, p.cache, 1, p.step, q, out, k, v, **args).run()
    assert torch.equal(p.cache.data.view(torch.uint8), kept.view(torch.uint8)) and torch.equal(out, want)
    if kind in (F16, BF16):
        assert torch.equal(out, want)
    rows.RopeAppend(table, p.cache, 1, p.step, q, q, k, v, **args).run()  # in place
    assert torch.equal(q, want) and torch.equal(p.cache.data.view(torch.uint8), kept.view(torch.uint8))


def test_append_positions():
    """the formula at the tokens' places, in the pages by the table"""
    heads, kv, dim, page = 4, 2, 64, 8
    lens, counts = [21, 9], [5, 2]
    p = Paged(F16, kv, dim, page, lens, counts)
    q, k, v = (_make((p.n, h, dim), F32, i) for i, h in enumerate((heads, kv, kv)))
    out, table = torch.empty_like(q), rows.RopeTable(dim, base=500000.0)
    rows.RopeAppend(table, p.cache, 0, p.step, q, out, k, v).run()
    pos = _ints([16, 17, 18, 19, 20, 7, 8])
    _near(out, *_want(table, q, pos, False, None, 0.0, 0.0), "q")
    wk, e = _want(table, k, pos, False, None, 0.0, 0.0)
    t = 0
    for i, (m, c) in enumerate(zip(lens, counts)):
        for at in range(m - c, m):
            slot = p.cache.data[0, :, p.rows[i][at // page], :, at % page]
            _near(slot[0][None], wk[t][None], e[t][None], "k")
            assert torch.equal(slot[1], v[t].half())
            t += 1
    assert (p.cache.data[1].view(torch.uint8) == 0x3A).all()  # (the other layer)


def test_rows_of_no_token():
    """behind the last sequence, of a sequence that takes no part or that the table does not know, past max_len, of an id that is no
    page: q's rows of no token and the pages stay as they are"""
    heads, kv, dim, page = 2, 2, 32, 8
    p = Paged(F16, kv, dim, page, [10, 12, 30, 9], [2, 2, 3, 2], live=[1, 0, 1, 1], extra=5, max_len=29)
    p.table[3, 1] = 10 ** 6  # (the fourth's second page)
    p.step.live[1] = 0
    n, table = p.n, rows.RopeTable(dim)
    q, k, v = (_make((n, h, dim), F32, i) for i, h in enumerate((heads, kv, kv)))
    out = torch.full_like(q, 5.0)
    rows.RopeAppend(table, p.cache, 0, p.step, q, out, k, v).run()
    pos = _ints([8, 9, 0, 0, 27, 28, 0, 7, 8] + [0] * 5)
    there = torch.tensor([1, 1, 0, 0, 1, 1, 0, 1, 1] + [0] * 5, dtype=torch.bool, device="cuda")
    want, e = _want(table, q, pos, False, None, 0.0, 0.0)
    _near(out[there], want[there], e[there], "q")
    assert (out[~there] == 5).all()
    written = (p.cache.data.view(torch.uint8) != 0x3A).view(2, 2, -1, kv, page, 2 * dim).any(-1)[0, 0].any(1)  # (page, slot)
    want_slots = {(p.rows[0][1], 0), (p.rows[0][1], 1), (p.rows[2][3], 3), (p.rows[2][3], 4), (p.rows[3][0], 7)}
    assert {tuple(x) for x in written.nonzero().tolist()} == want_slots
    p.step = attn.KvStep(p.step.start, p.step.len, p.table, n_tok=n, max_tok=3, max_len=30, seq=_ints([0, 9, -1, 1]))
    out.fill_(5.0)
    rows.RopeAppend(table, p.cache, 0, p.step, q, out, k, v).run()
    assert (out[2:7] == 5).all() and not (out[:2] == 5).any() and not (out[7:9] == 5).any()


def test_many_sequences():
    """more sequences than a wave reads at once"""
    seqs, heads, kv, dim, page = 150, 2, 1, 64, 16
    lens = [1 + (i * 37) % 90 for i in range(seqs)]
    p = Paged(BF16, kv, dim, page, lens, [1] * seqs)
    q, k, v = (_make((seqs, h, dim), BF16, i) for i, h in enumerate((heads, kv, kv)))
    out, want, table = torch.empty_like(q), torch.empty_like(q), rows.RopeTable(dim)
    rows.RopeAppend(table, p.cache, 1, p.step, q, out, k, v).run()
    rows.Rope(table, _ints([m - 1 for m in lens]), q, want).run()
    assert torch.equal(out, want)
    for i, m in enumerate(lens):
        assert torch.equal(p.cache.data[1, 1, p.rows[i][(m - 1) // page], :, (m - 1) % page], v[i])


def test_captured():
    heads, kv, dim = 8, 2, 128
    p = Paged(F16, kv, dim, 16, [50, 20], [1, 1])
    q, k, v = (_make((2, h, dim), F32, i) for i, h in enumerate((heads, kv, kv)))
    out, want, table = torch.empty_like(q), torch.empty_like(q), rows.RopeTable(dim)
    call = rows.RopeAppend(table, p.cache, 0, p.step, q, out, k, v)
    call.run()
    torch.cuda.synchronize()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        call.run(s.cuda_stream)
    for i in range(4):
        q.copy_(_make(q.shape, F32, 20 + i))
        p.step.len.copy_(_ints([50 - i, 20 - 2 * i]))  # (the replayed step goes by the lengths that it finds)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        rows.Rope(table, p.step.len - 1, q, want).run()
        assert torch.equal(out, want), i


def test_refusals():
    table = rows.RopeTable(32)
    q, k = _make((3, 4, 32), F32, 0), _make((3, 2, 32), F32, 1)
    pos = _ints([0, 1, 2])
    for args, kind in (((table, pos, q, q[:2]), ValueError), ((table, pos[:2], q, q), ValueError), ((table, pos, q, q, k), ValueError),
                       ((table, pos, q, q, k[:2], k[:2]), ValueError), ((table, pos, q, q, k.half(), k.half()), ValueError),
                       ((table, pos.long(), q, q), TypeError), ((table, pos, q.transpose(1, 2), q), TypeError), ((table, pos, q, q, k, k.half()), ValueError)):
        with pytest.raises(kind):
            rows.Rope(*args)
    with pytest.raises(RuntimeError):  # more rotary values than a head has
        rows.Rope(rows.RopeTable(64), pos, q, q).run()
    for bad in (dict(rot=33), dict(rot=0), dict(rot=32, base=0.5), dict(rot=32, scaling=dict(kind="more")), dict(rot=32, scaling=dict(kind="linear")),
                dict(rot=32, scaling=dict(kind="linear", factor=2.0, context=3)), dict(rot=32, scaling=dict(kind="linear", factor=0.0))):
        with pytest.raises(ValueError):
            rows.RopeTable(**bad)
    p = Paged(F16, 2, 32, 8, [9], [3])
    for bad in ((q, q, k[:2], k[:2]), (q, q, k, k.half()), (q, q[:2], k, k)):
        with pytest.raises(ValueError):
            rows.RopeAppend(table, p.cache, 0, p.step, *bad)
    with pytest.raises(RuntimeError):
        rows.RopeAppend(table, p.cache, 2, p.step, q, q, k, k).run()
    assert not capi.lib().osmos_rope(ctypes.byref(rows.Rope(table, pos, q, q).desc), None, None)
