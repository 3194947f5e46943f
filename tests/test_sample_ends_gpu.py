"""osmos_sample's rows end where they end: what stands before and behind a row's logits in memory, or in a last, partial piece of 16
bytes, is no token, whatever the limits' logits are. The rows are cut out of a larger tensor whose other values would change the
token or the count if they were taken. Tokens and counts are whole numbers, equal to the definition's; probabilities as
test_sample_gpu.py has them."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_sample_gpu import _check  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = [0.0, 0.3, 0.6, 0.9, 0.99]


def _inside(n, vocab, kind, around):
    """(n, vocab) rows in a tensor of `around`, 37 values before and 60 or more behind each, a whole row before and behind them all"""
    wide = torch.full((n + 2, vocab + 97 + (1 if kind == F32 else 0)), around, dtype=kind, device="cuda")
    return wide[1:n + 1, 37:37 + vocab]


@pytest.mark.parametrize("vocab", [1, 5, 1000, 1023, 2047])
def test_all_at_the_lowest_value(vocab):
    """float rows of the type's lowest value alone: all alike, in so few tokens that they are listed"""
    print(vocab, flush=True)
    low = torch.finfo(F32).min
    x = _inside(5, vocab, F32, low)
    got = _check(x, U, what="lowest", exact=True)
    assert got.tolist() == [min(vocab - 1, math.floor(float(torch.tensor(u)) * vocab)) for u in U]
    _check(x, U, top_p=[0.5] * 5, what="lowest, p", exact=True)
    _check(x, U, top_k=[300] * 5, what="lowest, k", exact=True)
    _check(x, U, min_p=[0.5] * 5, what="lowest, min-p", exact=True)


@pytest.mark.parametrize("kind", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("vocab", [1, 7, 1000, 2001])
def test_no_temperature_left(kind, vocab):
    """an infinite temperature: every token that can be chosen weighs the same"""
    print(kind, vocab, flush=True)
    x = _inside(5, vocab, kind, 2.0)
    x.copy_(torch.linspace(-3.0, 3.0, vocab, device="cuda").flip(0))
    x[1, ::2] = -math.inf
    x[2, 1::3] = math.nan
    x[3, :] = -math.inf
    x[4, vocab // 2:] = torch.finfo(kind).min
    for args in (dict(), dict(top_k=[5, 200, 3, 1, 900]), dict(top_p=[0.9] * 5), dict(min_p=[1.0] * 5)):
        got = _check(x, U, temperature=[math.inf] * 5, what="T inf %s" % args, exact=True, **args)
        assert int(got[3]) == -1


@pytest.mark.parametrize("kind,n", [(F32, 3), (F16, 3), (BF16, 3), (BF16, 300)], ids=str)
@pytest.mark.parametrize("warm", [True, False])
def test_long_rows_of_few_tokens(kind, n, warm):
    """rows of several slices (bf16's 300 counted by value) and of no whole number of pieces with 200 tokens that can be chosen: at the
    type's lowest value, or at an infinite temperature"""
    print(kind, n, warm, flush=True)
    vocab, low = 40009, torch.finfo(kind).min
    x = _inside(n, vocab, kind, 1.0 if warm else low)
    x.fill_(-math.inf)
    x[:, 100:40000:200] = 1.5 if warm else low
    x[:, vocab - 1] = 0.5 if warm else low
    u = [(i + 0.5) / n for i in range(n)]
    only = sorted({0, 1, n // 2, n - 2, n - 1})
    t = [math.inf if warm else 1.0] * n
    got = _check(x, u, temperature=t, what="few", exact=True, only=only)
    there = list(range(100, 40000, 200)) + [vocab - 1]
    assert got.tolist() == [there[math.floor(float(torch.tensor(v)) * len(there))] for v in u]
    _check(x, u, temperature=t, top_p=[0.7] * n, what="few, p", exact=True, only=only)
    _check(x, u, temperature=t, top_k=[50] * n, what="few, k", exact=True, only=only)
