"""Group normalisation with an activation, channels last: forward and gradients against 64 bits, and against differences."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}

# B, H, W, C, G: one value per group, odd channel counts (2-byte vectors), one channel per group, one group, a row that is one
# vector, slices that stay in registers (each class) and slices that take the passes, more than 512 vectors per row
SHAPES = [(1, 1, 1, 32, 32), (2, 3, 5, 33, 3), (3, 7, 7, 64, 64), (2, 9, 11, 40, 1), (1, 8, 8, 1280, 32), (2, 16, 16, 640, 32),
          (3, 32, 32, 320, 32), (2, 64, 64, 320, 32), (1, 40, 40, 960, 8), (1, 100, 90, 96, 1), (2, 5, 3, 9000, 2), (1, 3, 2, 1023, 1),
          (5, 1, 1, 4, 2), (1, 128, 128, 64, 32)]


def ops():
    from style_transfer_amd import ops as o
    return o


def make(B, H, W, C, dtype, seed, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((B, H, W, C), generator=g, device="cuda") * 1.5 + offset).to(dtype).permute(0, 3, 1, 2)
    w = 1 + 0.3 * torch.randn(C, generator=g, device="cuda")
    b = 0.3 * torch.randn(C, generator=g, device="cuda")
    dy = torch.randn((B, H, W, C), generator=g, device="cuda").to(dtype).permute(0, 3, 1, 2)
    return x, w, b, dy


def oracle(x, w, b, G, eps, act, dy=None):
    """64 bits; with dy also the gradients by the formula."""
    B, C = x.shape[:2]
    p = x.double().reshape(B, G, -1)
    mean, var = p.mean(-1, keepdim=True), p.var(-1, unbiased=False, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = ((p - mean) * rstd).reshape(x.shape)
    w64, b64 = (t.double().view(1, C, 1, 1) for t in (w, b))
    z = xh * w64 + b64
    s = torch.sigmoid(z)
    y = z * s if act == "silu" else z
    stat = (mean, rstd)
    if dy is None:
        return y, xh, stat
    dz = dy.double() * (s * (1 + z * (1 - s)) if act == "silu" else 1)
    dw, db = (dz * xh).sum((0, 2, 3)), dz.sum((0, 2, 3))
    dxh = dz * w64
    m = lambda t: t.reshape(B, G, -1).mean(-1, keepdim=True)
    ex = lambda t: t.expand(B, G, x[0].numel() // G).reshape(x.shape)
    dx = ex(rstd) * (dxh - ex(m(dxh)) - xh * ex(m(dxh * xh)))
    mags = ((dz * xh).abs().sum((0, 2, 3)), dz.abs().sum((0, 2, 3)), ex(rstd) * (dxh.abs() + ex(m(dxh.abs())) + xh.abs() * ex(m((dxh * xh).abs()))))
    return y, xh, stat, dx, dw, db, mags


# Longest chain of f32 additions behind a mean: rows of one thread (64), the tree over threads, chunks and channels.
CHAIN = 200


def xh_error(xh, stat, x, G):
    """The mean is off by CHAIN F32 of the group's mean magnitude, the standard deviation by as much relatively, and the
    subtraction and the product by one rounding each."""
    B = x.shape[0]
    mean, rstd = stat
    mag = x.double().abs().reshape(B, G, -1).mean(-1, keepdim=True)
    off = (CHAIN * F32 * mag * rstd).expand(B, G, x[0].numel() // G).reshape(x.shape)
    return off + (CHAIN + 4) * F32 * xh.abs()


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,W,C,G", SHAPES)
def test_forward_and_gradients(B, H, W, C, G, dtype, act):
    o = ops()
    x, w, b, dy = make(B, H, W, C, dtype, 7)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = o.group_norm_act(x, G, w, b, eps=1e-5, act=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(o.group_norm_act(x, G, w, b, eps=1e-5, act=act), y)
    assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32
    assert y.is_contiguous(memory_format=torch.channels_last) and dx.is_contiguous(memory_format=torch.channels_last)
    x, w, b = x.detach(), w.detach(), b.detach()
    Y, xh, stat, DX, DW, DB, (mw, mb, mx) = oracle(x, w, b, G, 1e-5, act, dy)
    ex = xh_error(xh, stat, x, G)
    W1, u = w.double().abs().view(1, C, 1, 1), HALF[dtype]
    z = (xh * w.double().view(1, C, 1, 1) + b.double().view(1, C, 1, 1)).abs()
    # |silu'| <= 1.1; the sigmoid of f32 exp and reciprocal is good to 8 F32 (+ the argument's rounding, |z| F32)
    ey = 1.1 * (ex * W1 + 4 * F32 * (z + 1)) + (8 + z) * F32 * z
    assert bool(((y.double() - Y).abs() <= ey + u * Y.abs() + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0)).all())
    # dz = dy act'(z), |act''| <= 0.5: off by 0.5 |dy| times z's error plus roundings; sums add CHAIN F32 of the magnitudes,
    # and a term's xh error counts where it is a factor
    edz = dy.double().abs() * (0.5 * (ex * W1 + 4 * F32 * (z + 1)) + (12 + z) * F32 if act == "silu" else torch.zeros_like(z))
    dzm = dy.double().abs() * 1.1
    assert bool(((dw.double() - DW).abs() <= (edz * xh.abs() + dzm * ex).sum((0, 2, 3)) + CHAIN * F32 * mw + 1e-30).all())
    assert bool(((db.double() - DB).abs() <= edz.sum((0, 2, 3)) + CHAIN * F32 * mb + 1e-30).all())
    gm = lambda t: t.reshape(B, G, -1).mean(-1, keepdim=True).expand(B, G, x[0].numel() // G).reshape(x.shape)
    rs = stat[1].expand(B, G, x[0].numel() // G).reshape(x.shape)
    a = edz * W1
    bnd = rs * (a + gm(a) + xh.abs() * gm(a * xh.abs() + dzm * W1 * ex) + ex * gm(dzm * W1 * xh.abs())) + (2 * CHAIN + 10) * F32 * mx
    assert bool(((dx.double() - DX).abs() <= bnd + u * DX.abs() + 1e-30 + (2.0 ** -25 if dtype == torch.float16 else 0)).all())


@pytest.mark.parametrize("H,W,C,G", [(6, 5, 12, 3), (70, 70, 32, 1), (3, 3, 7, 7)])
def test_gradients_against_differences(H, W, C, G):
    """Central differences of the kernel's own forward along random directions."""
    o = ops()
    x, w, b, dy = make(2, H, W, C, torch.float32, 11)
    y = o.group_norm_act(x.requires_grad_(True), G, w.requires_grad_(True), b.requires_grad_(True))
    grads = torch.autograd.grad(y, (x, w, b), dy)
    x, w, b = x.detach(), w.detach(), b.detach()
    h = 2.0 ** -7
    f = lambda a, c, e: float((o.group_norm_act(a, G, c, e).double() * dy.double()).sum())
    for i, gr in enumerate(grads):
        g = torch.Generator(device="cuda").manual_seed(30 + i)
        base = (x, w, b)
        v = torch.randn(base[i].shape, generator=g, device="cuda")
        v = v.contiguous(memory_format=torch.channels_last) if v.dim() == 4 else v
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + h * v, base[i] - h * v
        diff, want = (f(*up) - f(*dn)) / (2 * h), float((gr.double() * v.double()).sum())
        # truncation: h^2 / 6 of a third derivative of order one per term; rounding: F32 of each y (order one) over h
        mag = float(dy.double().norm()) * (1 + float(y.double().abs().max()))
        assert abs(diff - want) <= mag * (2 * h * h + 64 * F32 / h), (i, diff, want, mag)


def test_large_mean_keeps_its_digits():
    """Values 1000 +- 1: the centred sums keep the variance, in both forms."""
    o = ops()
    for shape in ((1, 16, 16, 64, 8), (1, 128, 128, 64, 2)):
        x, w, b, _ = make(*shape[:4], torch.float32, 3, offset=1000.0)
        got = o.group_norm_act(x, shape[4], w, b, act="none")
        Y, xh, stat = oracle(x, w, b, shape[4], 1e-5, "none")
        ex = xh_error(xh, stat, x, shape[4])
        assert bool(((got.double() - Y).abs() <= (ex + 4 * F32 * (xh.abs() + 1)) * w.double().abs().view(1, -1, 1, 1) + 4 * F32 * Y.abs()).all())


def test_tokens_without_affine_and_cast_parameters():
    o = ops()
    x = torch.randn(3, 77, 48, device="cuda", dtype=torch.bfloat16)
    y = o.group_norm_act(x, 6, act="none", eps=1e-6)
    Y, _, _ = oracle(x.permute(0, 2, 1).unsqueeze(-1), torch.ones(48, device="cuda"), torch.zeros(48, device="cuda"), 6, 1e-6, "none")
    Y = Y[..., 0].permute(0, 2, 1)
    assert bool(((y.double() - Y).abs() <= 2.0 ** -8 * Y.abs() + 300 * F32 * (1 + Y.abs())).all())
    w = torch.randn(48, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    z = o.group_norm_act(x, 6, w, None)
    (gw,) = torch.autograd.grad(z.float().sum(), (w,))
    assert gw.dtype == torch.bfloat16 and torch.isfinite(gw).all()
    only = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(o.group_norm_act(only, 6).float().square().sum(), (only,))
    assert gx.shape == x.shape and torch.isfinite(gx.float()).all()


@pytest.mark.parametrize("H,C,G", [(16, 320, 32), (100, 96, 2)])
def test_unaligned_storage(H, C, G):
    """A tensor that starts between vector boundaries, in both forms."""
    o = ops()
    x, w, b, dy = make(2, H, H, C, torch.bfloat16, 5)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    odd = flat[1:].view(2, H, H, C)
    odd.copy_(x.permute(0, 2, 3, 1))
    odd = odd.permute(0, 3, 1, 2)
    res = []
    for t in (x.clone(memory_format=torch.preserve_format), odd):
        t = t.detach().requires_grad_(True)
        y = o.group_norm_act(t, G, w, b)
        res.append((y,) + torch.autograd.grad(y, (t,), dy))
    for a, c in zip(*res):
        # the same numbers summed in another order: at most a rounding of the stored type apart
        assert bool(((a.double() - c.double()).abs() <= 2.0 ** -7 * a.double().abs() + 1e-4).all())


def test_results_repeat_and_captured_training_step():
    o = ops()
    x, w, b, dy = make(2, 32, 32, 64, torch.bfloat16, 9)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = o.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(torch.randn_like(x) + i)
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(out, step()):
            assert torch.equal(a, c)


def test_another_stream_while_the_first_is_busy():
    o = ops()
    x, w, b, _ = make(2, 100, 100, 96, torch.float32, 4)
    want = o.group_norm_act(x, 2, w, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(o.group_norm_act(x, 2, w, b))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in outs)


def test_second_derivative_is_refused():
    """create_graph gives the gradients; differentiating them again is an error, not a silent zero."""
    x = torch.randn(2, 6, 8, device="cuda:0", requires_grad=True)
    w = torch.randn(8, device="cuda:0", requires_grad=True)
    y = ops().group_norm_act(x, 2, w)
    want = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    got = torch.autograd.grad(y, (x, w), torch.ones_like(y), create_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        got[0].square().sum().backward()


def test_gradient_in_another_order_or_type():
    """An incoming gradient that is expanded, strided or of another type gives what its contiguous copy gives."""
    torch.manual_seed(9)
    x = torch.randn(2, 6, 5, 8, device="cuda:0").permute(0, 3, 1, 2).requires_grad_()
    y = ops().group_norm_act(x, 4)
    g = torch.randn(2, 8, 6, 5, device="cuda:0")
    want = torch.autograd.grad(y, x, g.contiguous(memory_format=torch.channels_last), retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, x, g, retain_graph=True)[0], want)
    one = torch.ones((), device="cuda:0").expand(2, 8, 6, 5)
    want = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, x, one, retain_graph=True)[0], want)


@pytest.mark.parametrize("B,H,W,C,G", [(1, 8, 8, 64, 4), (2, 8, 8, 64, 4), (1, 100, 90, 96, 1), (2, 70, 64, 320, 8)])
def test_only_some_gradients(B, H, W, C, G):
    """Weight's, bias's or the input's gradient alone is what it is among all three (one image and several, in registers and by
    passes)."""
    x, w, b, dy = make(B, H, W, C, torch.float32, 5)
    every = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops().group_norm_act(every[0], G, *every[1:]), every, dy)
    for i in range(3):
        some = [t.detach().requires_grad_(k == i) for k, t in enumerate(every)]
        got = torch.autograd.grad(ops().group_norm_act(some[0], G, *some[1:]), some[i], dy)[0]
        assert torch.equal(got, want[i])
