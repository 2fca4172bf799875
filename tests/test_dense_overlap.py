"""CPU: which buffers eas.ops takes for overlapping, against the sets of their elements."""

import random

from easy_as_b200.ops import _Rows, _share


def elements(r):
    return {r.ptr + 2 * (i * r.ld + j) for i in range(r.rows) for j in range(r.cols)}


def test_rows_that_share_no_element():
    """Never told apart wrongly; and told apart always where both lie in one pitch, or one is a single row."""
    rng = random.Random(1)
    apart = 0
    for _ in range(20000):
        ld = rng.randint(1, 12)
        a, b = (_Rows(0x1000 + 2 * rng.randint(0, 40), rng.randint(1, 5), rng.randint(1, ld), ld, (), None) for _ in range(2))
        if rng.random() < 0.2:
            b.ld = rng.randint(b.cols, 15)
        truth = bool(elements(a) & elements(b))
        lo, hi = a.ptr, a.ptr + a.span()
        meet = b.ptr < hi and lo < b.ptr + b.span()
        said = meet and _share(a, b)
        assert said or not truth
        if a.ld == b.ld or a.rows == 1 or b.rows == 1:
            if not truth and meet:
                apart += 1
            # a row longer than the gap between two rows wraps: that is told as an overlap where they meet at all
            long = (a.rows == 1 and a.cols > b.ld) or (b.rows == 1 and b.cols > a.ld)
            assert said == truth or long, (a.ptr, a.rows, a.cols, a.ld, b.ptr, b.rows, b.cols, b.ld)
    assert apart > 500
