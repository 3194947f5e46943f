"""osmos_sample's `kept` under a min_p so small that its border lies among tokens that add nothing to any sum: those of at least min_p
times the greatest weight, by the definition in float64 (test_sample_gpu.py's)."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_sample_gpu import _check  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MIN_P = [1e-14, 1e-20, 1e-30, 1e-45, 3e-14, 1e-13]  # (by turns; the bins' last weight is some 4e-14)


def _rows(n, vocab, kind):
    """a great token and 3000 around 2^-43 to 2^-47 of its weight, 300 further down by powers of ten, the others at e^-60 and, of every second
    row, masked by the type's lowest value or by -infinity"""
    x = torch.full((n, vocab), -60.0, device="cuda")
    x[:, 7] = 0.0
    x[:, 100:3100] = -29.4 - 1.1e-3 * torch.arange(3000, device="cuda")
    x[:, 3200:3500] = -33.0 - 0.25 * torch.arange(300, device="cuda")
    x = x.to(kind)
    x[1::2, 3500::2] = torch.finfo(kind).min
    x[1::2, 3501::4] = -math.inf
    return x


@pytest.mark.parametrize("kind,n,vocab", [(F32, 6, 4000), (F16, 6, 4000), (BF16, 6, 4000), (F32, 6, 40009), (F16, 6, 40009), (BF16, 6, 40009),
                                          (BF16, 300, 40009)], ids=str)
def test_least_weights(kind, n, vocab):
    print(kind, n, vocab, flush=True)
    x, only = _rows(n, vocab, kind), list(range(6)) + ([n - 2, n - 1] if n > 6 else [])
    u = [(i + 0.5) / n for i in range(n)]
    min_p = [MIN_P[i % 6] for i in range(n)]
    each = lambda *v: [v[i % len(v)] for i in range(n)]  # noqa: E731
    got = _check(x, u, min_p=min_p, what="min-p", exact=True, only=only)
    assert got.tolist() == [7] * n
    for i in (0, 1):  # (every min_p on masked rows and on others)
        _check(x.roll(i, 0), u, min_p=min_p, what="min-p, rolled %d" % i, exact=True, only=only)
    _check(x, u, min_p=min_p, top_k=each(40, 3200, 1500, 3001, 1000, 2), what="k, min-p", exact=True, only=only)
    _check(x, u, min_p=min_p, top_k=each(3500, vocab - 1, 3100, 1024, 1025, vocab), what="far k, min-p", exact=True, only=only)
    _check(x, u, min_p=min_p, top_p=each(0.5, 0.999999, 1.0, 0.9), what="p, min-p", exact=True, only=only)
    _check(x, u, min_p=min_p, temperature=each(1.0, 0.5, 2.0, 0.9), what="T, min-p", exact=True, only=only)


def test_nothing_but_the_greatest_in_the_bins():
    """few tokens asked for, most of them of no weight"""
    for vocab in (50, 33000):
        x = torch.full((4, vocab), -60.0, device="cuda")  # (8.8e-27)
        x[:, 3] = 0.0
        x[:, 9] = -40.0  # (4.2e-18)
        x[2:, 20:] = torch.finfo(F32).min
        u = [0.1, 0.5, 0.9, 0.99]
        for min_p in (1e-17, 1e-25, 1e-26, 1e-27, 1e-44):
            _check(x, u, min_p=[min_p] * 4, top_k=[40] * 4, what="k, %g" % min_p, exact=True)
            _check(x, u, min_p=[min_p] * 4, what="%g" % min_p, exact=True)


def test_far_logits():
    """the border past the type's lowest value, and where logits are so far apart that no other token is in the bins"""
    x = torch.full((5, 3000), -3.0e38, device="cuda")
    x[:, 1::2] = torch.finfo(F32).min
    x[:, 2999] = -2.9e38
    x[3:] *= 1e-30
    for t in (1.0, 1e36, 1e37, 1e38):
        _check(x, [0.0, 0.2, 0.4, 0.6, 0.8], temperature=[t] * 5, min_p=[1e-14, 1e-30, 1e-44, 1e-14, 1e-30], what="T %g" % t, exact=True)
