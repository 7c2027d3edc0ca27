"""Shared-prefix attention, on 16-bit keys and on codes, within bounds that tests/test_shared_attn_bounds_host.py shows to leave
no room for a lost key range, a misplaced scale or a causal limit that is off by one."""
import pytest
import torch

from shared_attn_bounds import BF16, CASES, CODES, F16, Case

pytestmark = pytest.mark.gpu


def ops():
    from style_transfer_amd import ops as o
    return o


def check(c, got):
    out, av, qk, vm = c.exact("cuda")
    over = (got.double() - out).abs() / c.tolerance(out, av, qk, vm)
    assert float(over.max()) <= 1, (float(over.max()), int((over > 1).sum()), (over > 1).nonzero()[:3].tolist())


@pytest.mark.parametrize("name", list(CASES))
def test_within_the_bounds(name):
    c = Case(**CASES[name])
    got = c.run(ops())
    check(c, got)
    for _ in range(2):                                   # sums have one order: the same bits every time
        assert torch.equal(c.run(ops()), got)


@pytest.mark.parametrize("fmt", CODES + [("none", "none")])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_sequence_alone_and_in_a_batch(dtype, fmt):
    """Both decompositions, six sequences at once and each by itself, are as near to the exact result."""
    kw = dict(Hq=4, Hkv=2, n=1, P=600, S=40, d=64, dtype=dtype, fmt=fmt)
    c = Case(B=6, lens=[40, 1, 0, 33, 17, 40], **kw)
    check(c, c.run(ops()))
    for b in range(6):
        one = Case(B=1, lens=[c.lens[b]], **kw)
        one.q = c.q[b:b + 1]
        for x in ("k", "v", "ks", "vs"):
            if hasattr(c.own, x):
                setattr(one.own, x, getattr(c.own, x)[b:b + 1].contiguous())
        check(one, one.run(ops()))
