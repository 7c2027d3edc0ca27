"""The 8-bit key/value cache: rows against their definition in 64 bits, positions, padding, strides, odd values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TOP = {"int8": 127.0, "e4m3": 448.0}
F32 = 2.0 ** -24                       # half a step of float32, relative


def ops():
    from style_transfer_amd import ops as o
    return o


def rand(shape, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype).cuda()


def check_rows(x, codes, scale, fmt):
    """x (rows, d), codes as float64 numbers, scale: one row at a time by the definition."""
    x64, top = x.double(), TOP[fmt]
    amax = x.abs().float().amax(-1)
    want = torch.where(amax >= 2.0 ** -100, (amax.double() / top).float(), torch.zeros_like(amax))       # rounded once
    assert torch.equal(scale, want)
    live = want > 0
    z = x64[live] / (amax[live].double() / top).unsqueeze(-1)
    err = (codes[live] - z).abs()
    # the nearest code is half a step away at most; the quotient top / amax and the product are rounded once each (2 F32 relative)
    if fmt == "int8":
        step = torch.ones_like(z)
    else:
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
        step = step.clamp_min(2.0 ** -9)
    assert bool((err <= step / 2 * (1 + 1e-9) + 4 * F32 * z.abs()).all()), float((err / step).max())
    assert bool((codes[~live] == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,n,d,S", [(1, 1, 1, 8, 1), (3, 8, 7, 40, 20), (2, 5, 33, 80, 40), (16, 8, 1, 64, 9), (1, 3, 129, 256, 130),
                                       (2, 2, 65, 136, 65)])
def test_rows_by_the_definition(B, H, n, d, S, dtype, fmt):
    o = ops()
    cache = o.kv_cache(B, H, S, d, fmt)
    k, v = rand((B, H, n, d), 1, dtype), rand((B, H, n, d), 2, dtype)
    start = torch.tensor([(3 * b) % (S - n + 1) for b in range(B)], dtype=torch.int32, device="cuda")
    o.kv_cache_write(cache, k, v, start)
    got = o.kv_cache_read(cache, start, n, torch.float32)
    for x, codes, scale, out in ((k, cache.k_codes, cache.k_scale, got[0]), (v, cache.v_codes, cache.v_scale, got[1])):
        for b in range(B):
            s = int(start[b])
            c, f = codes[b, :, s:s + n].float().double(), scale[b, :, s:s + n]
            check_rows(x[b].reshape(-1, d), c.reshape(-1, d), f.reshape(-1), fmt)
            # read back: code * scale, exact in 64 bits, rounded once to float32
            assert torch.equal(out[b], (c * f.double().unsqueeze(-1)).float())
            # everything else is as it was
            rest = torch.ones(S, dtype=torch.bool, device="cuda")
            rest[s:s + n] = False
            assert int(codes[b][:, rest].view(torch.uint8).sum()) == 0 and float(scale[b][:, rest].abs().sum()) == 0
    for t in (torch.bfloat16, torch.float16):
        kk, vv = o.kv_cache_read(cache, start, n, t)
        assert torch.equal(kk, got[0].to(t)) and torch.equal(vv, got[1].to(t))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_strides_padding_and_the_ends(fmt):
    o = ops()
    B, H, n, d, S = 4, 8, 6, 40, 10
    wide = rand((B, n, 2 * H, d), 3, torch.bfloat16)
    k, v = wide[:, :, :H].transpose(1, 2), wide[:, :, H:].transpose(1, 2)       # two halves of one projection
    start = torch.tensor([0, 7, -2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    length = torch.tensor([4, 6, 6, 6], dtype=torch.int32, device="cuda")
    cache, dense = o.kv_cache(B, H, S, d, fmt), o.kv_cache(B, H, n, d, fmt)
    o.kv_cache_write(cache, k, v, start, length)
    o.kv_cache_write(dense, k.contiguous(), v.contiguous())
    written = {0: (0, 0, 4), 1: (7, 0, 3), 2: (0, 2, 4)}                         # sequence: (position, first row, rows)
    for name in ("k_codes", "k_scale", "v_codes", "v_scale"):
        a, b = (getattr(c, name).view(torch.uint8 if "codes" in name else torch.float32) for c in (cache, dense))
        want = torch.zeros_like(a)
        for s, (at, first, rows) in written.items():
            want[s, :, at:at + rows] = b[s, :, first:first + rows]
        assert torch.equal(a, want), name
    kk, _ = o.kv_cache_read(cache, start, n, torch.float32)                      # outside the cache: zeros
    assert float(kk[3].abs().sum()) == 0 and float(kk[2, :, :2].abs().sum()) == 0 and float(kk[1, :, 3:].abs().sum()) == 0
    assert float(kk[2, :, 2:].abs().sum()) > 0
    # rows that start between 16-byte boundaries are copied first
    odd = rand((B, H, n, d + 1), 4, torch.bfloat16)[..., 1:]
    two = [o.kv_cache(B, H, n, d, fmt) for _ in range(2)]
    o.kv_cache_write(two[0], odd, odd)
    o.kv_cache_write(two[1], odd.contiguous(), odd.contiguous())
    assert torch.equal(two[0].k_codes.view(torch.uint8), two[1].k_codes.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_odd_values(fmt):
    o = ops()
    rows = torch.zeros((1, 1, 9, 16))
    rows[0, 0, 1, 3] = float("inf")
    rows[0, 0, 2, 15] = float("nan")
    rows[0, 0, 3] = 2.0 ** -101                       # below the smallest row that is kept
    rows[0, 0, 4, 0], rows[0, 0, 4, 1] = 3e38, -3e38
    rows[0, 0, 5] = 2.0 ** -100
    rows[0, 0, 6, :2] = torch.tensor([1.0, -1.0])
    rows[0, 0, 7] = -0.0
    rows[0, 0, 8] = torch.linspace(-1, 1, 16)
    cache = o.kv_cache(1, 1, 9, 16, fmt)
    o.kv_cache_write(cache, rows.cuda(), rows.cuda())
    out = o.kv_cache_read(cache, 0, 9, torch.float32)[0][0, 0].cpu()
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    for i in (0, 3, 7):
        assert (out[i] == 0).all() and float(cache.k_scale[0, 0, i]) == 0
    # the largest magnitude maps to the largest code: amax / top * top, two roundings
    for i, a in ((4, 3e38), (5, 2.0 ** -100), (6, 1.0)):
        assert abs(float(out[i, 0]) / a - 1) <= 3 * F32
    assert torch.equal(out[6, :2], torch.stack([out[6, 0], -out[6, 0]]))


def test_no_rows_and_int_positions():
    o = ops()
    cache = o.kv_cache(2, 3, 5, 24)
    e = torch.empty((2, 3, 0, 24), device="cuda")
    o.kv_cache_write(cache, e, e, 1)
    k, v = o.kv_cache_read(cache, 2, 0)
    assert k.shape == v.shape == (2, 3, 0, 24) and float(cache.k_scale.abs().sum()) == 0
    x = rand((2, 3, 2, 24), 5)
    o.kv_cache_write(cache, x, -x, 3)
    k, v = o.kv_cache_read(cache, 3, 2, torch.float32)
    assert torch.equal(k, -v) and float((k - x).abs().max()) <= float(x.abs().max()) / 127 * 0.51


def test_offsets_beyond_32_bits():
    o = ops()
    H, S, d = 9, 1 << 20, 256                           # 2.4e9 codes: the last head starts behind 2^31
    cache = o.kv_cache(1, H, S, d)
    x = rand((1, H, 3, d), 6, torch.bfloat16)
    start = torch.tensor([S - 3], dtype=torch.int32, device="cuda")
    o.kv_cache_write(cache, x, 2 * x, start)
    k, v = o.kv_cache_read(cache, start, 3, torch.float32)
    check_rows(x[0, -1], cache.k_codes[0, -1, -3:].double(), cache.k_scale[0, -1, -3:], "int8")
    assert torch.equal(2 * k, v)
    assert int(cache.k_codes[0, 0, :4].abs().sum()) == 0 and int(cache.k_codes[0, -1, -4].abs().sum()) == 0


def test_captured_steps_append():
    """A captured step appends one token per replay: the position lives on the device."""
    o = ops()
    B, H, d, S = 3, 4, 64, 8
    caches = [o.kv_cache(B, H, S, d, "e4m3") for _ in range(2)]
    steps = [rand((B, H, 1, d), 20 + i, torch.bfloat16) for i in range(S)]
    slot, pos = steps[0].clone(), torch.zeros(B, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        o.kv_cache_write(caches[0], slot, slot, pos)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o.kv_cache_write(caches[0], slot, slot, pos)
    torch.cuda.synchronize()
    for i in range(S):
        slot.copy_(steps[i])
        pos.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        o.kv_cache_write(caches[1], steps[i], steps[i], i)
        for n in ("k_codes", "v_codes"):
            assert torch.equal(getattr(caches[0], n).view(torch.uint8), getattr(caches[1], n).view(torch.uint8)), i
        assert torch.equal(caches[0].k_scale, caches[1].k_scale)
