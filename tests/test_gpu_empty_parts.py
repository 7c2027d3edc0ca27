"""Caches without positions, and attention with an empty prefix or empty own parts: they add nothing, in any form and at any
head_dim."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    from style_transfer_amd import ops as o
    return o


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("B,S", [(2, 0), (0, 3)])
def test_empty_cache(B, S, fmt):
    o = ops()
    cache = o.kv_cache(B, 3, S, 8, fmt)
    x = torch.randn(B, 3, 4, 8, device="cuda")
    o.kv_cache_write(cache, x, x)
    o.kv_cache_write(cache, x[:, :, :0], x[:, :, :0], torch.zeros(B, dtype=torch.int32, device="cuda"))
    for n in (0, 5):
        k, v = o.kv_cache_read(cache, 0, n, torch.float16)
        assert k.shape == v.shape == (B, 3, n, 8) and k.dtype == torch.float16
        assert float(k.abs().sum()) == float(v.abs().sum()) == 0


@pytest.mark.parametrize("fmt", ["none", "int8", "e4m3"])
@pytest.mark.parametrize("d", [8, 16, 40, 136])
@pytest.mark.parametrize("n", [1, 70])
def test_empty_parts(n, d, fmt):
    o = ops()
    g = torch.Generator(device="cuda").manual_seed(d)
    r = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16)

    def part(B, keys):
        if fmt == "none":
            k, v = r(B, 2, keys, d), r(B, 2, keys, d)
            return (k, v) if B > 1 else (k[0], v[0])
        cache = o.kv_cache(B, 2, keys, d, fmt)
        o.kv_cache_write(cache, r(B, 2, keys, d), r(B, 2, keys, d))
        return cache

    q, pre, own = r(3, 4, n, d), part(1, 33), part(3, 9)
    assert torch.equal(o.shared_prefix_attention(q, part(1, 0), own), o.shared_prefix_attention(q, None, own))
    assert torch.equal(o.shared_prefix_attention(q, pre, part(3, 0)), o.shared_prefix_attention(q, pre, None))
    lens = torch.tensor([0, 5, -1], dtype=torch.int32, device="cuda")
    assert torch.equal(o.shared_prefix_attention(q, pre, part(3, 0), own_len=lens, causal=True), o.shared_prefix_attention(q, pre, None))
    none = o.shared_prefix_attention(q, part(1, 0), part(3, 0), own_len=lens)
    assert none.shape == (3, n, 4 * d) and float(none.abs().sum()) == 0
