"""Group norm on tensors of more than 2^31 values: the last image's values and gradients."""
import pytest
import torch

import test_gpu_group_norm as base

pytestmark = pytest.mark.gpu


def make(B, H, W, C, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, dy = (torch.randn((B, H, W, C), generator=g, device="cuda", dtype=torch.bfloat16).permute(0, 3, 1, 2) for _ in range(2))
    w = 1 + 0.3 * torch.randn(C, generator=g, device="cuda")
    return x, w, 0.3 * torch.randn(C, generator=g, device="cuda"), dy


def step(x, w, b, dy, G, act):
    x = x.detach().requires_grad_()
    y = base.ops().group_norm_act(x, G, w, b, act=act)
    return y.detach(), torch.autograd.grad(y, x, dy)[0]


def test_slices_in_registers():
    """4200 images: the last one has the bits that it has alone (the form does not depend on the batch)."""
    x, w, b, dy = make(4200, 32, 32, 512, 1)
    assert x.numel() > 2 ** 31
    whole = step(x, w, b, dy, 32, "silu")
    for i in (0, 4095, 4199):
        for a, c in zip(whole, step(x[i:i + 1], w, b, dy[i:i + 1], 32, "silu")):
            assert torch.equal(a[i:i + 1], c)


def test_by_passes():
    """Two images of 1.1 million rows, the last group of the last one against 64 bits.  A thread joins 270 batches of 8 rows:
    2000 F32 for the longest chain."""
    G, chain = 32, 2000
    x, w, b, dy = make(2, 1100, 1000, 1024, 2)
    assert x.numel() > 2 ** 31
    y, dx = (t[1:, -32:] for t in step(x, w, b, dy, G, "none"))
    x, dy, w, b = x[1:, -32:].double(), dy[1:, -32:].double(), w[-32:].double(), b[-32:].double()
    Y, xh, (mean, rstd), DX, _, _, (_, _, mx) = base.oracle(x, w, b, 1, 1e-5, "none", dy)
    W1 = w.abs().view(1, -1, 1, 1)
    ex = chain * base.F32 * x.abs().mean() * rstd.item() + (chain + 4) * base.F32 * xh.abs()
    u = 2.0 ** -8
    assert bool(((y.double() - Y).abs() <= ex * W1 + 4 * base.F32 * (xh.abs() * W1 + 1) + u * Y.abs()).all())
    g = dy.abs() * W1
    bound = rstd.item() * (xh.abs() * (g * ex).mean() + ex * (g * xh.abs()).mean()) + (2 * chain + 10) * base.F32 * mx
    assert bool(((dx.double() - DX).abs() <= bound + u * DX.abs()).all())
