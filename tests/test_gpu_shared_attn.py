"""Shared-prefix attention against its definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ops():
    from style_transfer_amd import ops as o
    return o


def randn(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def reference(q, prefix, own, lens, causal, scale):
    """q (B, Hq, n, d); prefix (kp, vp) float64 (Hkv, P, d); own float64 (B, Hkv, S, d).  -> out, and for the tolerance the
    largest |v| a row sees and the largest sum |q_i k_i| scale over its keys."""
    B, Hq, n, d = q.shape
    Hkv = prefix[0].shape[0]
    out = torch.zeros((B, n, Hq, d), dtype=torch.float64, device=q.device)
    vmax = torch.zeros((B, n, Hq, 1), dtype=torch.float64, device=q.device)
    qk = torch.zeros((B, n, Hq, 1), dtype=torch.float64, device=q.device)
    for b in range(B):
        L = min(max(int(lens[b]), 0), own[0].shape[2])
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            k = torch.cat([prefix[0][hk], own[0][b, hk, :L]])
            v = torch.cat([prefix[1][hk], own[1][b, hk, :L]])
            if not len(k):
                continue
            P = len(k) - L
            s = q[b, h].double() @ k.T * scale
            if causal:
                i = torch.arange(n, device=q.device)[:, None]
                s = s.masked_fill(torch.arange(len(k), device=q.device)[None] >= P + (L - n + 1 + i).clamp_min(0), -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[b, :, h] = p @ v
            vmax[b, :, h] = v.abs().max()
            qk[b, :, h] = (q[b, h].double().abs() @ k.abs().T).amax(-1, keepdim=True) * scale
    return out.reshape(B, n, Hq * d), vmax.expand(B, n, Hq, d).reshape(B, n, Hq * d), qk.expand(B, n, Hq, d).reshape(B, n, Hq * d)


def tolerance(ref, vmax, qk, dtype, quantised):
    """Half a step u of the 16-bit type: each probability is off by u and so may be their sum (2 u of the largest value), the
    output is rounded once (u).  Keys and values that were codes are rounded to the type too: a logit is then off by u sum|q k|,
    a weight by twice that (exponentially), a value by u.  f32 logits and exponentials: 2^-18 of sum|q k|, and 2^-18.  A half's
    probabilities below 2^-30 of the largest are lost: 2^-20 for all keys of a test together."""
    u = HALF[dtype]
    delta = 2 * qk * ((u if quantised else 0) + 2.0 ** -18)
    return vmax * (torch.expm1(delta) + 2 * u + (u if quantised else 0) + 2.0 ** -18 + 2.0 ** -20) + u * ref.abs()


def fill(o, fmt, t, n_keys, seed, dtype, shape):
    """A part as the operator takes it, and its numbers in 64 bits."""
    k, v = randn(shape, seed, dtype), randn(shape, seed + 1, dtype)
    if fmt == "none":
        return (k, v), (k.double(), v.double())
    four = shape if len(shape) == 4 else (1,) + shape
    cache = o.kv_cache(four[0], four[1], four[2], four[3], fmt)
    o.kv_cache_write(cache, k.view(four), v.view(four))
    num = lambda c, s: (c.float().double() * s.double().unsqueeze(-1)).view(shape)
    return cache, (num(cache.k_codes, cache.k_scale), num(cache.v_codes, cache.v_scale))


def run(B, Hq, Hkv, n, P, S, d, dtype, fmt=("none", "none"), causal=False, lens=None, scale=None, seed=0, qscale=1.0):
    o = ops()
    q = randn((B, n, Hq, d), seed, dtype, qscale).transpose(1, 2)
    pre, pre64 = fill(o, fmt[0], None, P, seed + 10, dtype, (Hkv, P, d)) if P else (None, (torch.zeros((Hkv, 0, d), dtype=torch.float64, device="cuda"),) * 2)
    own, own64 = fill(o, fmt[1], None, S, seed + 20, dtype, (B, Hkv, S, d)) if S else (None, (torch.zeros((B, Hkv, 0, d), dtype=torch.float64, device="cuda"),) * 2)
    own_len = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = o.shared_prefix_attention(q, pre, own, own_len=own_len, causal=causal, scale=scale)
    sc = d ** -0.5 if scale is None else scale
    ref, vmax, qk = reference(q, pre64, own64, [S] * B if lens is None else lens, causal, sc)
    tol = tolerance(ref, vmax, qk, dtype, fmt != ("none", "none"))
    err = (got.double() - ref).abs()
    bad = err > tol
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol.clamp_min(1e-30)).max()), bad.nonzero()[:3].tolist())
    return got


TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 48, 56, 64, 72, 80, 96, 104, 128, 136, 160, 168, 192, 224, 256])
def test_head_dims(d, dtype):
    run(2, 2, 1, 1, 70, 33, d, dtype, lens=[33, 5])                 # rows of the batch together, waves share the keys
    run(1, 2, 2, 150, 65, 40, d, dtype)                             # many rows: waves share the rows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Hq,Hkv,n,P,S", [
    (1, 1, 1, 1, 1, 0), (1, 1, 1, 1, 0, 1), (1, 8, 8, 1, 31, 0), (4, 8, 2, 1, 33, 1), (3, 4, 4, 1, 0, 257), (33, 4, 1, 1, 1000, 3),
    (5, 14, 2, 3, 129, 64), (2, 8, 8, 64, 100, 100), (2, 4, 2, 65, 64, 63), (1, 8, 8, 128, 0, 128), (2, 2, 2, 129, 1, 1),
    (1, 4, 4, 257, 63, 65), (2, 16, 2, 17, 500, 77), (70, 8, 8, 1, 300, 20), (1, 1, 1, 1, 5000, 4000), (2, 2, 2, 300, 2000, 1500),
])
def test_shapes(B, Hq, Hkv, n, P, S, dtype):
    run(B, Hq, Hkv, n, P, S, 40, dtype)
    run(B, Hq, Hkv, n, P, S, 128, dtype, seed=1)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n", [1, 5, 40, 200])
@pytest.mark.parametrize("P", [0, 45])
def test_ragged_and_empty_rows(P, n, causal):
    """No own keys, fewer own keys than queries, lengths outside the tensor: rows without keys give zeros."""
    lens = [0, 1, 3, n, 97, 64, -5, 1000]
    got = run(8, 4, 2, n, P, 97, 64, torch.bfloat16, causal=causal, lens=lens)
    if P == 0:
        assert float(got[0].abs().sum()) == 0 and float(got[6].abs().sum()) == 0


@pytest.mark.parametrize("fmt", [("int8", "int8"), ("e4m3", "e4m3"), ("int8", "none"), ("none", "e4m3")])
@pytest.mark.parametrize("B,Hq,Hkv,n,d", [(4, 8, 2, 1, 128), (3, 4, 4, 5, 80), (1, 8, 8, 200, 40), (40, 4, 2, 1, 64)])
def test_cached_keys(B, Hq, Hkv, n, d, fmt):
    for dtype in TYPES:
        run(B, Hq, Hkv, n, 333, 70, d, dtype, fmt=fmt, causal=n > 1, lens=[70 - 3 * (b % 20) for b in range(B)])


@pytest.mark.parametrize("d", [8, 16, 24, 40, 72, 136, 168, 256])
def test_cached_keys_of_every_row_width(d):
    """Rows of 8 (mod 16) codes, whose last sixteen overlap; a cache that ends with the last row."""
    for n in (1, 130):
        run(2, 2, 2, n, 45, 37, d, torch.bfloat16, fmt=("int8", "e4m3"), lens=[37, 20])


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits_and_rising_keys(dtype):
    """Logits that keep growing along the keys: the softmax reference moves many times, in every tile and split."""
    o = ops()
    d, P = 64, 700
    q = torch.ones((2, 2, 1, d), device="cuda", dtype=dtype)
    k = (torch.arange(P, device="cuda", dtype=torch.float32)[None, :, None] * 0.25).expand(2, P, d).to(dtype).contiguous()
    v = randn((2, P, d), 3, dtype)
    for n in (1, 140):
        qq = q.expand(2, 2, n, d).contiguous()
        got = o.shared_prefix_attention(qq, (k, v))
        ref, vmax, qk = reference(qq, (k.double(), v.double()), (torch.zeros((2, 2, 0, d), dtype=torch.float64, device="cuda"),) * 2, [0, 0], False, d ** -0.5)
        assert bool(((got.double() - ref).abs() <= tolerance(ref, vmax, qk * 0 + 30, dtype, False)).all())
    run(3, 4, 2, 1, 400, 50, 80, dtype, qscale=12.0, lens=[50, 0, 9])
    run(1, 2, 2, 140, 400, 50, 80, dtype, qscale=12.0)


@pytest.mark.parametrize("n,G", [(1, 4), (6, 1), (40, 2), (300, 1)])
def test_what_is_masked_does_not_matter(n, G):
    """Infinities and NaN behind own_len, and in keys that the causal order hides from some rows, reach none of those."""
    o = ops()
    B, Hkv, P, S, d = 2, 2, 50, 400, 40
    q = randn((B, Hkv * G, n, d), 1, torch.bfloat16)
    pre = (randn((Hkv, P, d), 2, torch.bfloat16), randn((Hkv, P, d), 3, torch.bfloat16))
    own = [randn((B, Hkv, S, d), s, torch.bfloat16) for s in (4, 5)]
    lens = torch.tensor([380, 333], dtype=torch.int32, device="cuda")
    want = o.shared_prefix_attention(q, pre, tuple(own), own_len=lens, causal=True)
    for x, bad in ((0, float("nan")), (1, float("nan")), (1, float("inf")), (0, -float("inf"))):
        dirty = [t.clone() for t in own]
        for b in range(B):
            dirty[x][b, :, int(lens[b]):] = bad
        assert torch.equal(o.shared_prefix_attention(q, pre, tuple(dirty), own_len=lens, causal=True), want)
        # the last token's value: only the last query of a sequence sees it
        for b in range(B):
            dirty[x][b, :, int(lens[b]) - 1, 7] = bad
        got = o.shared_prefix_attention(q, pre, tuple(dirty), own_len=lens, causal=True)
        assert torch.equal(got[:, :-1], want[:, :-1])
        if bad != -float("inf"):
            last = got[:, -1].reshape(B, Hkv * G, d)
            assert not torch.isfinite(last[:, :, 7]).any()


def test_strides_and_prefix_len():
    o = ops()
    B, H, n, P, S, d = 2, 4, 3, 90, 21, 40
    packed = randn((B, n, 3, H, d), 1, torch.float16)
    q = packed[:, :, 1].transpose(1, 2)                              # a slice of a joint projection
    kv = randn((P + 7, 2, H, d), 2, torch.float16)
    pre = (kv[:P, 0].transpose(0, 1), kv[:P, 1].transpose(0, 1))     # tokens first, heads inside
    ow = randn((S, B, H, d), 3, torch.float16)
    own = (ow.permute(1, 2, 0, 3), ow.permute(1, 2, 0, 3))
    want = o.shared_prefix_attention(q.contiguous(), tuple(t.contiguous() for t in pre), tuple(t.contiguous() for t in own))
    assert torch.equal(o.shared_prefix_attention(q, pre, own), want)
    longer = (kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1))
    assert torch.equal(o.shared_prefix_attention(q, longer, own, prefix_len=P), want)
    odd = randn((H, P, d + 3), 5, torch.float16)[..., 3:]            # rows between 16-byte boundaries: copied first
    assert torch.equal(o.shared_prefix_attention(q, (odd, odd), own), o.shared_prefix_attention(q, (odd.contiguous(),) * 2, own))
    none = o.shared_prefix_attention(q, pre, prefix_len=0)
    assert none.shape == (B, n, H * d) and float(none.abs().sum()) == 0
    given = torch.full((B, n, H * d), 9.0, dtype=torch.float16, device="cuda")
    assert o.shared_prefix_attention(q, pre, own, out=given) is given and torch.equal(given, want)


def test_one_head_position_independent_of_the_batch():
    """A sequence's result does not depend on who else is in the batch beyond the order of f32 sums."""
    o = ops()
    q = randn((6, 4, 1, 64), 1, torch.bfloat16)
    pre = (randn((2, 600, 64), 2, torch.bfloat16), randn((2, 600, 64), 3, torch.bfloat16))
    all_ = o.shared_prefix_attention(q, pre)
    for b in range(6):
        one = o.shared_prefix_attention(q[b:b + 1], pre)
        assert bool(((one.double() - all_[b:b + 1].double()).abs() <= 4 * 2.0 ** -8 * float(pre[1].abs().max())).all())


def test_offsets_beyond_32_bits():
    """Own keys whose sequences lie more than 2^31 bytes apart."""
    o = ops()
    B, H, S, d = 2, 9, 1 << 20, 128
    k = torch.zeros((B, H, S, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    L = [5, S]
    k[1, -1, -1] = 4.0
    v[1, -1, -1] = 3.0
    v[0, :, :5] = 1.0
    q = torch.ones((B, H, 1, d), dtype=torch.bfloat16, device="cuda")
    out = o.shared_prefix_attention(q, None, (k, v), own_len=torch.tensor(L, dtype=torch.int32, device="cuda")).view(B, H, d)
    w = math.exp(4 * 128 ** 0.5 - 0)
    want = 3.0 * w / (w + S - 1)
    assert bool(((out[1, -1].double() - want).abs() <= 4 * 2.0 ** -8 * 3).all()) and bool((out[0].double() == 1).all())


def test_graph_replays_follow_the_device_lengths():
    """A captured decoding step: append to the 8-bit cache, attend; the lengths live on the device."""
    o = ops()
    B, Hq, Hkv, d, P, S = 3, 8, 2, 64, 200, 40
    pre = o.kv_cache(1, Hkv, P, d)
    o.kv_cache_write(pre, randn((1, Hkv, P, d), 1, torch.bfloat16), randn((1, Hkv, P, d), 2, torch.bfloat16))
    caches = [o.kv_cache(B, Hkv, S, d) for _ in range(2)]
    steps = [[randn((B, 1, h, d), 50 + 3 * i + j, torch.bfloat16).transpose(1, 2) for j, h in enumerate((Hq, Hkv, Hkv))] for i in range(5)]
    q, k, v = (t.clone() for t in steps[0])
    pos = torch.tensor([0, 3, 30], dtype=torch.int32, device="cuda")
    first, lens = pos.clone(), pos + 1

    def step(cache, q, k, v):
        o.kv_cache_write(cache, k, v, pos)
        return o.shared_prefix_attention(q, pre, cache, own_len=lens)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], q, k, v)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(caches[0], q, k, v)
    torch.cuda.synchronize()
    for i, (a, b, c) in enumerate(steps):
        q.copy_(a), k.copy_(b), v.copy_(c)
        pos.copy_(first + i)
        lens.copy_(pos + 1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(caches[1], a, b, c)), i


def test_streams_do_not_share_scratch():
    o = ops()
    q = randn((4, 8, 1, 64), 1, torch.bfloat16)
    pre = (randn((8, 4000, 64), 2, torch.bfloat16), randn((8, 4000, 64), 3, torch.bfloat16))
    want = o.shared_prefix_attention(q, pre)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(o.shared_prefix_attention(q, pre))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in outs)


@pytest.mark.parametrize("fmt", [("none", "none"), ("int8", "int8"), ("none", "e4m3")])
@pytest.mark.parametrize("d", [24, 40, 56, 64])
def test_many_rows_on_a_full_chip(d, fmt):
    """Enough rows for 512 workgroups of 256: a wave keeps two tiles of queries.  Row tails, grouped heads, ragged lengths, the
    causal order, and the keys of a prefix split in two."""
    dtype = TYPES[d // 8 % 2]
    run(32, 16, 16, 150, 77, 40, d, dtype, fmt=fmt, causal=True, lens=[(7 * b) % 43 - 1 for b in range(32)])
    run(64, 16, 8, 70, 65, 0, d, dtype, fmt=fmt)
    run(16, 16, 16, 131, 1100, 0, d, dtype, fmt=fmt)
