"""The bounds that shared-prefix attention is held to tell a right result from a wrong one: mistakes are planted in the 64-bit
form, on the CPU, and have to leave the bounds.  (bf16, whose bounds are the wider ones.)"""
import pytest

from shared_attn_bounds import BF16, CASES, Case


@pytest.mark.parametrize("name", [n for n, c in CASES.items() if c["dtype"] == BF16])
def test_mistakes_leave_the_bounds(name):
    c = Case(**CASES[name])
    out, av, qk, vm = c.exact()
    tol, seen = c.tolerance(out, av, qk, vm), av > 0

    def outside(wrong):
        return float((((wrong - out).abs() > tol) & seen).sum()) / int(seen.sum())

    assert outside(out) == 0
    assert outside(0 * out) > 0.9
    if c.P:
        assert outside(c.exact(drop=("prefix", 0, c.P // 2))[0]) > 0.4
        if c.P < 500:
            assert outside(c.exact(drop=("prefix", max(0, c.P - 32), c.P))[0]) > 0.01
    if c.S:
        assert outside(c.exact(drop=("own", 0, c.S))[0]) > 0.3
    if c.fmt[0] != "none" or c.S and c.fmt[1] != "none":
        assert outside(c.exact(shifted=True)[0]) > 0.2
    if c.causal:
        for late in (1, -1):
            assert outside(c.exact(late=late)[0]) > 0.01
