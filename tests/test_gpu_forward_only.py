"""Shared-prefix attention has no backward pass: a gradient that is asked for is an error, never silently missing."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from style_transfer_amd import ops as o
    return o


def tensors(dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device=DEV).to(dtype)
    return r(2, 4, 3, 40), (r(2, 33, 40), r(2, 33, 40)), (r(2, 2, 9, 40), r(2, 2, 9, 40))


@pytest.mark.parametrize("which", range(5))
def test_backward_raises(which):
    """Whichever input asks for a gradient: the forward result is as ever, the backward pass an error."""
    o = ops()
    q, pre, own = tensors()
    want = o.shared_prefix_attention(q, pre, own)
    assert not want.requires_grad
    k, v = own
    (q, *pre, k, v)[which].requires_grad_()
    got = o.shared_prefix_attention(q, tuple(pre), (k, v))
    assert got.requires_grad and torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError, match="forward only"):
        got.float().sum().backward()
    with pytest.raises(RuntimeError, match="out="):
        o.shared_prefix_attention(q, tuple(pre), (k, v), out=torch.empty_like(want))
    with torch.no_grad():
        given = torch.empty_like(want)
        assert o.shared_prefix_attention(q, tuple(pre), (k, v), out=given) is given and torch.equal(given, want)


def test_attention_module_on_codes():
    """The network's layer behind an 8-bit entry: a training step through its queries is refused, its output layer alone
    trains."""
    from style_transfer_amd.attention import CrossAttention
    o = ops()
    torch.manual_seed(3)
    attn = CrossAttention(80, heads=2, dim_head=40).to(DEV)
    attn.cnt_name = "/nowhere/img.jpg"
    x, rows = torch.randn(2, 9, 80, device=DEV), torch.randn(1, 2, 33, 40, device=DEV)
    kv = o.kv_cache(1, 2, 33, 40, "int8", DEV)
    o.kv_cache_write(kv, rows, -rows)
    call = lambda m: m(x, k_injected=kv, v_injected=kv, injection_config={"T": 1.5, "gamma": 0.5})
    with torch.no_grad():
        want = call(attn)
    assert torch.equal(call(attn).detach(), want)
    with pytest.raises(RuntimeError, match="forward only"):
        call(attn).sum().backward()
    frozen = copy.deepcopy(attn)
    frozen.to_q.requires_grad_(False)
    call(frozen).sum().backward()
    assert torch.isfinite(frozen.to_out[0].weight.grad).all() and float(frozen.to_out[0].weight.grad.abs().sum()) > 0


def test_pairs_of_any_kind():
    """A pair may be a tuple, a list, a stacked tensor or an iterator, with gradients tracked or not."""
    o = ops()
    q, pre, own = tensors()
    want = o.shared_prefix_attention(q, pre, own)
    for make in (list, torch.stack, iter):
        assert torch.equal(o.shared_prefix_attention(q, make(pre), make(own)), want)
        with torch.no_grad():
            assert torch.equal(o.shared_prefix_attention(q, make(pre), make(own)), want)
    pre[1].requires_grad_()
    assert o.shared_prefix_attention(q, iter(pre), own).requires_grad
