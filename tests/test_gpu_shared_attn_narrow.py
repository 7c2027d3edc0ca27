"""Shared-prefix attention on codes of head_dim 8, which the kernel takes as rows of 16: within the same bounds as every other
head_dim (keys exact), with each argument in its place."""
import pytest
import torch

from shared_attn_bounds import BF16, CODES, F16, Case
from test_gpu_shared_attn_bounds import check, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", CODES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kw", [dict(B=3, Hq=4, Hkv=2, n=1, P=500, S=60, lens=[60, 0, 7]), dict(B=2, Hq=7, Hkv=1, n=31, P=300, S=150, causal=True),
                                dict(B=1, Hq=2, Hkv=2, n=200, P=400, S=0), dict(B=5, Hq=2, Hkv=1, n=2, P=0, S=90)])
def test_within_the_bounds(kw, dtype, fmt):
    c = Case(d=8, dtype=dtype, fmt=fmt, qscale=2.0, **kw)
    check(c, c.run(ops()))


@pytest.mark.parametrize("own_fmt", ["int8", "none"])
def test_arguments_keep_their_meaning(own_fmt):
    o = ops()
    c = Case(B=2, Hq=4, Hkv=2, n=3, P=80, S=20, d=8, dtype=F16, fmt=("int8", own_fmt), lens=[20, 4])
    q, pre, own, lens = c.q.cuda(), c.pre.on_gpu(o), c.own.on_gpu(o), torch.tensor(c.lens, dtype=torch.int32, device="cuda")
    want = o.shared_prefix_attention(q, pre, own, own_len=lens)
    assert torch.equal(o.shared_prefix_attention(q, pre, own, own_len=lens, scale=8 ** -0.5), want)
    given = torch.full_like(want, 9.0)
    assert o.shared_prefix_attention(q, pre, own, own_len=lens, out=given) is given and torch.equal(given, want)
    short = o.QuantKV(*(t[:, :, :50].contiguous() for t in pre.tensors()))
    assert torch.equal(o.shared_prefix_attention(q, pre, own, own_len=lens, prefix_len=50), o.shared_prefix_attention(q, short, own, own_len=lens))
    for bad in (given[:, :, :16], given.float(), given[:1]):
        with pytest.raises(ValueError, match="out must be"):
            o.shared_prefix_attention(q, pre, own, own_len=lens, out=bad)
    with pytest.raises(ValueError):
        o.shared_prefix_attention(q, o.kv_cache(1, 2, 9, 16), own)
    with pytest.raises(ValueError):
        o.shared_prefix_attention(q, o.kv_cache(2, 2, 9, 8), own)
