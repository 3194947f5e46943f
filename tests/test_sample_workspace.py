"""osmos_sample_workspace's sizes, and the calls refused without one (no GPU: refused calls read nothing)."""
import ctypes

from libosmos_amd import capi
from tests.test_rows_checks import A, _sample

R = ctypes.byref
BINS, LIST = 1024, 2048  # a slice's bins (a sum and a count each), a row's listed tokens


def _need(**o):
    return capi.lib().osmos_sample_workspace(R(_sample(**o)))


def test_sizes():
    long = dict(vocab=1 << 20, stride=1 << 20)
    one = _need(n=1, probs=None, **long)
    # (slices of 16384 tokens; a row's prefix sums and its list)
    assert one >= (1 << 20) // 16384 * BINS * 12 + BINS * 12 + LIST * 8
    assert _need(n=8, probs=None, **long) >= 8 * (one - 1024) and _need(n=8, **long) > _need(n=8, probs=None, **long)
    assert _need(vocab=1000, probs=None) == 0 and _need(vocab=1000) > 0  # (a short row's probabilities alone)
    assert one % 256 == 0 and _need(n=3, **long) % 256 == 0 and _need(n=3) % 256 == 0


def test_a_call_without():
    L = capi.lib()
    for d in (_sample(n=1, vocab=1 << 20, stride=1 << 20), _sample(n=3, vocab=40000, stride=40000, type=30), _sample()):
        need = L.osmos_sample_workspace(R(d))
        assert need > 0
        for ws, size in ((None, need), (None, 1 << 40), (A, need - 1), (A, 0), (A + 64, need), (A + 64, 1 << 40)):
            assert not L.osmos_sample(R(d), ctypes.c_void_p(ws), size, None)
