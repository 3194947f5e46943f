"""osmos_rope_turns' YaRN at its ends, by the checks' library of test_rows_checks.py (no GPU): pairs that make `slow` turns or less in the
context are divided by the factor, those of `fast` or more stay, whatever the context's length."""
import math

import pytest

from tests.test_rows_checks import H, _turns  # noqa: F401


@pytest.mark.parametrize("rot", [2, 8, 20, 64, 128, 256])
@pytest.mark.parametrize("slow,fast", [(1.0, 32.0), (0.5, 0.75), (4.0, 5.0), (100.0, 1000.0)])
def test_yarn_ends(H, rot, slow, fast):  # noqa: F811
    plain, _ = _turns(H, rot)
    for context in (1.0, 3.0, 6.2, 6.4, 12.0, 25.0, 40.0, 512.0, 8192.0, 1e6, 1e9, 1e12):
        yarn, _ = _turns(H, rot, 3, factor=16.0, context=context, low=slow, high=fast)
        for i, (a, b) in enumerate(zip(yarn, plain)):
            n, note = context * b, (context, i)
            assert b / 16 * (1 - 1e-13) <= a <= b * (1 + 1e-13), note
            if n < slow * (1 - 1e-9):
                assert math.isclose(a, b / 16, rel_tol=1e-13), note
            if n > fast * (1 + 1e-9):
                assert math.isclose(a, b, rel_tol=1e-13), note
