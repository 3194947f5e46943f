"""osmos_rope at far positions against whole-number arithmetic: position x turns[i] is formed exactly (float64 turns are whole numbers of
powers of two), its fraction rounded once to float64. A pair (1, 0) turns into the angle's cosine and sine themselves.

What a sine or cosine may be off by: the quarter's angle to float, at most pi / 4: 2^-25; a sine's last step, of results up to 0.71:
2^-25, its term -x^3 / 6 (up to 0.081, two products rounded before it): 2^-26.6, that term's own coefficient sum: 2^-28, the series' first
term left out: 2^-29; 2^-23.6 in all. A cosine's last step: 2^-25, the square's rounding times 0.45: 2^-26.1, the sum that it is
multiplied by: 2^-26.7, the angle's rounding times 0.71: 2^-25.5; 2^-23.6 too. The fraction itself adds 2^-50."""
import math
from fractions import Fraction

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from libosmos_amd import attn, rows  # noqa: E402

F32, F16 = torch.float32, torch.float16
OFF = 2.0 ** -23.5


def _turned(turns, positions):
    """cosines and sines (positions, pairs) in float64"""
    c, s = [], []
    for p in positions:
        f = [float(Fraction(t) * p % 1) * (2 * math.pi) for t in turns]
        c.append([math.cos(x) for x in f])
        s.append([math.sin(x) for x in f])
    return torch.tensor(c, dtype=torch.float64), torch.tensor(s, dtype=torch.float64)


def _run(table, positions, pairs):
    n, rot = len(positions), table.rot
    q = torch.zeros((n, 1, 64), device="cuda")
    at = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    q[..., at[0]] = 1.0
    out = torch.empty_like(q)
    rows.Rope(table, torch.tensor(positions, dtype=torch.int32, device="cuda"), q, out, pairs=pairs).run()
    out = out[:, 0].cpu().double()
    return out[:, at[0]], out[:, at[1]]


def _check(table, positions, pairs):
    want = _turned(table.turns.tolist(), positions)
    for got, w, what in zip(_run(table, positions, pairs), want, ("cosine", "sine")):
        off = (got - w).abs()
        assert float(off.max()) <= OFF, "%s off by 2^%.2f at position %d" % (what, math.log2(float(off.max())), positions[int(off.max(1).values.argmax())])


FAR = [0, 1, -1, 3, 131071, -(2 ** 24) - 1, 2 ** 30 + 77, 2 ** 31 - 1, -(2 ** 31), 1999999999, -1888888888, 2 ** 31 - 129]


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("first", [0, 2 ** 24, 2 ** 30, 2 ** 31 - 2048, -(2 ** 31)])
def test_far_rows(first, pairs):
    _check(rows.RopeTable(8), [first + i for i in range(2048)], pairs)


@pytest.mark.parametrize("turns", [[0.7310585786300049, 0.4999999999999999, 1 / 3, 1.0 - 2.0 ** -53], [1000.1, -333.3333, 123456.789, 2.0 ** -30],
                                   [4194303.3, -2097151.77, 2.0 ** 20 + 1 / 7, 5e-324]], ids=str)
def test_tables_of_any_turns(turns):
    """a table of one's own, to 2^53 turns in all"""
    table = rows.RopeTable(8)
    table.turns.copy_(torch.tensor(turns, dtype=torch.float64))
    _check(table, FAR, False)
    _check(table, [2 ** 31 - 1 - 7919 * i for i in range(500)], True)


def test_far_turns_are_the_table():
    """against the definition's base^(-2 i / rot) radians: what the table's rounding to float64 adds, in turns: the power, its quotient by 2 pi
    and that number itself by half a step each, the power one step more: 2.5 x 2^-52 of the turns in all"""
    table, p = rows.RopeTable(64, base=10000.0), 2 ** 31 - 1
    c, s = _run(table, [p], False)
    # (2 pi to 60 digits)
    two_pi = Fraction(6283185307179586476925286766559005768394338798750211641949889, 10 ** 60)
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    for i in range(32):
        turn = Fraction(Decimal(10000) ** (Decimal(-2 * i) / Decimal(64))) / two_pi
        f = float(turn * p % 1) * 2 * math.pi
        more = 2.5 * 2.0 ** -52 * float(turn) * p * 2 * math.pi
        assert abs(float(c[0, i]) - math.cos(f)) <= OFF + more and abs(float(s[0, i]) - math.sin(f)) <= OFF + more, i


def test_far_append():
    """the cache's rows by the same angles: the bits of osmos_rope at these positions"""
    n, page, most = 5, 1024, 2 ** 19
    cache = attn.KvCache.empty(F16, 1, most // page + 1, 1, page, 16)
    start, length = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, n], [most - 3]))
    table = torch.arange(most // page, dtype=torch.int32, device="cuda")[None].contiguous()
    step = attn.KvStep(start, length, table, n_tok=n, max_tok=n, max_len=most)
    turns = rows.RopeTable(8)
    turns.turns.copy_(torch.tensor([4099.123456789, 0.1, 77777.7, 1e-9], dtype=torch.float64))
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    q, k, v = (torch.randn((n, 1, 16), generator=g, device="cuda") for _ in "qkv")
    out, want, half = torch.empty_like(q), torch.empty_like(q), torch.empty((n, 1, 16), dtype=F16, device="cuda")
    rows.RopeAppend(turns, cache, 0, step, q, out, k, v).run()
    pos = torch.arange(most - 3 - n, most - 3, dtype=torch.int32, device="cuda")
    rows.Rope(turns, pos, q, want).run()
    rows.Rope(turns, pos, k, half).run()
    assert torch.equal(out, want) and torch.equal(cache.data[0, 0, -2, 0, page - 3 - n:page - 3], half[:, 0])
    c, s = _turned(turns.turns.tolist(), pos.tolist())
    a, b = (x[:, 0].cpu().double() for x in q.split(4, 2)[:2])
    y = torch.cat((a * c - b * s, b * c + a * s), 1)
    e = (a.abs() + b.abs()) * 2.0 ** -21  # (as test_rope_gpu.py)
    assert ((out[:, 0, :8].cpu().double() - y).abs() <= torch.cat((e, e), 1)).all()
