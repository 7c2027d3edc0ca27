"""Group norm whose input needs no gradient: that of its weights alone is computed, and has the bits that it has beside the
input's."""
import pytest
import torch

from test_gpu_group_norm import make

pytestmark = pytest.mark.gpu


def ops():
    from style_transfer_amd import ops as o
    return o


# one image and several in registers, by passes with joined chunks, by passes with a join of their own (a row wider than 512
# vectors of its element)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,H,W,C,G", [(1, 8, 8, 64, 4), (3, 9, 7, 40, 5), (2, 100, 90, 96, 1), (2, 60, 60, 1023, 3)])
def test_weights_alone(B, H, W, C, G, dtype):
    x, w, b, dy = make(B, H, W, C, dtype, 5)
    xs, ws, bs = (t.detach().clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, w, b))
    want = torch.autograd.grad(ops().group_norm_act(xs, G, ws, bs), (xs, ws, bs), dy)[1:]
    for kw, kb in ((True, True), (True, False), (False, True)):
        ws, bs = w.detach().requires_grad_(kw), b.detach().requires_grad_(kb)
        leaves = [t for t in (ws, bs) if t.requires_grad]
        got = torch.autograd.grad(ops().group_norm_act(x, G, ws, bs), leaves, dy)
        for g, t in zip(got, [t for t, k in zip(want, (kw, kb)) if k]):
            assert torch.equal(g, t)


def test_no_gradient_of_the_input_is_made():
    """Neither computed nor allocated: the backward pass of 64 MB takes less than that."""
    x, w, b, dy = make(4, 128, 128, 512, torch.bfloat16, 6)
    size = x.numel() * 2
    w.requires_grad_()
    y = ops().group_norm_act(x, 32, w, b)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    (dw,) = torch.autograd.grad(y, w, dy)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < size // 2 and torch.isfinite(dw).all()
