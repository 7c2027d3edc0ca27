"""Refusals of the 8-bit cache, shared-prefix attention and group norm: argument checks come before any GPU call."""
import pytest
import torch

from style_transfer_amd import lib, ops

A = 1 << 20                 # an aligned address that nothing reads


def st(*v):
    return lib.strides3(*v)


def code(rc):
    return rc, lib.load().sid_last_error().decode()


def write(B=1, H=2, n=3, S=4, d=40, dtype=0, fmt=1, k=A, codes=A, start=A, ks=None):
    ks = st(H * n * d, n * d, d) if ks is None else ks
    return code(lib.load().sid_kv_cache_write(k, A, ks, ks, codes, A, A, A, start, None, B, H, n, S, d, dtype, fmt, None))


def read(B=1, H=2, n=3, S=4, d=40, dtype=0, fmt=1, out=A, codes=A):
    return code(lib.load().sid_kv_cache_read(codes, A, A, A, out, A, A, B, H, n, S, d, dtype, fmt, None))


@pytest.mark.parametrize("kw,text", [
    (dict(d=41), "head_dim"), (dict(d=0), "head_dim"), (dict(d=264), "head_dim"), (dict(S=0), ">= 1"), (dict(B=0), ">= 1"),
    (dict(fmt=0), "format"), (dict(fmt=3), "format"), (dict(dtype=3), "dtype"), (dict(n=-1), "negative"), (dict(k=None), "NULL"),
    (dict(k=A + 8), "16-byte"), (dict(codes=A + 4), "8-byte"), (dict(start=None), "NULL"), (dict(ks=st(240, 121, 40)), "16-byte"),
    (dict(B=300, H=300), "too many"), (dict(B=1, H=1000, n=2 ** 31 - 1), "too many rows")])
def test_cache_write_refusals(kw, text):
    rc, msg = write(**kw)
    assert rc == -22 and text in msg, (rc, msg)


@pytest.mark.parametrize("kw,text", [(dict(d=4), "head_dim"), (dict(fmt=0), "format"), (dict(dtype=-1), "dtype"), (dict(n=-1), "negative"),
                                     (dict(out=None), "NULL"), (dict(out=A + 8), "16-byte"), (dict(codes=A + 4), "8-byte"),
                                     (dict(n=2 ** 31 - 1, d=256), "too large")])
def test_cache_read_refusals(kw, text):
    rc, msg = read(**kw)
    assert rc == -22 and text in msg, (rc, msg)


def test_nothing_to_do_is_no_error():
    assert write(n=0)[0] == 0 and read(n=0)[0] == 0


def source(k=A, fmt=0, stride=(640, 320, 40), scale=None):
    return lib.kv_source(k, A, scale or 0, scale or 0, *stride, *stride, 16, 8, fmt)


def attend(q=A, B=1, Hq=4, Hkv=2, n=1, d=40, P=8, S=0, scale=1.0, dtype=1, pre=None, own=None, ws=A, ws_bytes=1 << 30, qs=(160, 40, 160), out=A):
    pre = source() if pre is None else pre
    ref = lambda s: s or None
    return code(lib.load().sid_shared_attn_fwd(q, st(*qs), ref(pre), ref(own), None, out, B, Hq, Hkv, n, d, P, S, scale, 0, dtype,
                                               ws, ws_bytes, None))


@pytest.mark.parametrize("kw,text", [
    (dict(Hq=5), "divide"), (dict(d=20), "head_dim"), (dict(d=264), "head_dim"), (dict(dtype=0), "bf16 or f16"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(q=None), "NULL"),
    (dict(q=A + 8), "16-byte"), (dict(qs=(160, 41, 160)), "16-byte"), (dict(n=0), ">= 1"), (dict(P=-1), "negative"), (dict(out=A + 2), "8-byte"),
    (dict(pre=0), "NULL"), (dict(S=8), "own part"), (dict(pre=source(k=A + 8)), "aligned"), (dict(pre=source(stride=(0, 321, 40))), "aligned"),
    (dict(pre=source(stride=(0, 320, -40))), "distance"), (dict(pre=source(stride=(0, 320, 1 << 24))), "distance"),
    (dict(pre=source(fmt=1)), "scales"), (dict(d=8, pre=source(fmt=1, scale=A), qs=(32, 8, 32)), "16 or more"), (dict(pre=source(fmt=4)), "format"), (dict(P=1 << 30), "too many"), (dict(B=1 << 23), "too many")])
def test_shared_attention_refusals(kw, text):
    rc, msg = attend(**kw)
    assert rc == -22 and text in msg, (rc, msg)


def test_shared_attention_workspace():
    L = lib.load()
    need = L.sid_shared_attn_workspace_bytes(4, 8, 8, 1, 64, 8000, 100, 0)
    assert need > 256
    src = source(stride=(0, 8000 * 64, 64))
    rc, msg = attend(B=4, Hq=8, Hkv=8, d=64, P=8000, S=100, pre=src, own=source(stride=(51200, 6400, 64)), ws_bytes=need - 1, qs=(512, 64, 512))
    assert rc == -12 and str(need) in msg
    rc, msg = attend(B=4, Hq=8, Hkv=8, d=64, P=8000, S=100, pre=src, own=source(stride=(51200, 6400, 64)), ws=A + 64, qs=(512, 64, 512))
    assert rc == -22 and "256-byte" in msg
    assert L.sid_shared_attn_workspace_bytes(1, 8, 8, 4096, 40, 4096, 0, 0) >= 256
    # parts held differently are walked by items of their own, whose results are joined
    assert L.sid_shared_attn_workspace_bytes(4, 8, 8, 4096, 40, 4096, 4096, 1) > L.sid_shared_attn_workspace_bytes(4, 8, 8, 4096, 40, 4096, 4096, 0)
    assert L.sid_shared_attn_workspace_bytes(1, 8, 3, 1, 40, 8, 0, 0) == 0


def norm(x=A, B=1, N=4, C=64, G=8, eps=1e-5, act=1, dtype=0, ws=A, ws_bytes=1 << 30, mean=A):
    return code(lib.load().sid_group_norm_act_fwd(x, A, A, A, mean, A, B, N, C, G, eps, act, dtype, ws, ws_bytes, None))


def norm_bwd(x=A, B=1, N=4, C=64, G=8, act=1, dtype=0, ws=A, ws_bytes=1 << 30, dy=A):
    return code(lib.load().sid_group_norm_act_bwd(dy, x, A, A, A, A, A, A, A, B, N, C, G, act, dtype, ws, ws_bytes, None))


@pytest.mark.parametrize("kw,text", [(dict(G=7), "divide"), (dict(C=0), ">= 1"), (dict(B=65536), "too large"), (dict(act=2), "activation"),
                                     (dict(dtype=3), "dtype"), (dict(x=None), "NULL")])
def test_group_norm_refusals(kw, text):
    for f in (norm, norm_bwd):
        rc, msg = f(**kw)
        assert rc == -22 and text in msg, (rc, msg)


def test_group_norm_refusals_of_one_direction():
    assert norm(eps=-1.0)[0] == -22 and norm(eps=float("nan"))[0] == -22 and norm(mean=None)[0] == -22 and norm_bwd(dy=None)[0] == -22
    assert norm_bwd(ws=None)[0] == -22 and norm_bwd(ws=A + 16)[0] == -22
    L = lib.load()
    need = L.sid_group_norm_workspace_bytes(1, 1 << 20, 64, 8, 0, 0)
    assert norm(N=1 << 20, ws_bytes=256)[0] == -12 and need > 256
    assert L.sid_group_norm_workspace_bytes(1, 4, 64, 7, 0, 0) == 0
    assert norm(x=A + 2)[0] == -22                                     # not aligned to its elements


def test_python_layer_refuses_what_is_not_on_a_gpu():
    x = torch.zeros(1, 2, 3, 40)
    cache = ops.kv_cache(1, 2, 4, 40, device="cpu")
    for f in (lambda: ops.kv_cache_write(cache, x, x), lambda: ops.kv_cache_read(cache, 0, 2),
              lambda: ops.shared_prefix_attention(x.bfloat16(), (x[0].bfloat16(), x[0].bfloat16())),
              lambda: ops.group_norm_act(torch.zeros(1, 4, 8), 2)):
        with pytest.raises(RuntimeError, match="GPU memory"):
            f()


def test_python_layer_refuses_wrong_shapes_and_types():
    z = torch.zeros
    cache = ops.kv_cache(2, 2, 4, 40, device="cpu")
    x = z(2, 2, 3, 40)
    bad = [
        (ValueError, lambda: ops.kv_cache(1, 1, 1, 12, device="cpu")),
        (ValueError, lambda: ops.kv_cache(1, 1, 1, 16, fmt="int4", device="cpu")),
        (TypeError, lambda: ops.QuantKV(z(1, 1, 2, 8), z(1, 1, 2), z(1, 1, 2, 8), z(1, 1, 2))),
        (ValueError, lambda: ops.QuantKV(z(1, 1, 2, 8).to(torch.int8), z(1, 1, 3), z(1, 1, 2, 8).to(torch.int8), z(1, 1, 2))),
        (RuntimeError, lambda: ops.QuantKV(z(1, 2, 2, 8).to(torch.int8).transpose(1, 2), z(1, 2, 2), z(1, 2, 2, 8).to(torch.int8), z(1, 2, 2))),
        (ValueError, lambda: ops.kv_cache_write(cache, x, x[:, :, :2])),
        (ValueError, lambda: ops.kv_cache_write(cache, x[:1], x[:1])),
        (TypeError, lambda: ops.kv_cache_write(cache, x.double(), x.double())),
        (ValueError, lambda: ops.kv_cache_write(cache, x, x, z(2, dtype=torch.int64))),
        (ValueError, lambda: ops.kv_cache_write(cache, x, x, z(3, dtype=torch.int32))),
        (ValueError, lambda: ops.kv_cache_read(cache, 0, -1)),
        (TypeError, lambda: ops.kv_cache_read(cache, 0, 1, torch.int8)),
        (ValueError, lambda: ops.shared_prefix_attention(z(2, 3, 40).bfloat16())),
        (TypeError, lambda: ops.shared_prefix_attention(x)),
        (ValueError, lambda: ops.group_norm_act(z(1, 8, 4, 4), 2)),                              # not channels last
        (ValueError, lambda: ops.group_norm_act(z(1, 8), 2)),
        (ValueError, lambda: ops.group_norm_act(z(1, 4, 8), 2, act="gelu")),
        (ValueError, lambda: ops.group_norm_act(z(1, 4, 8), 2, z(7))),
        (TypeError, lambda: ops.group_norm_act(z(1, 4, 8, dtype=torch.float64), 2)),
    ]
    for err, f in bad:
        with pytest.raises(err):
            f()


def test_rows_are_copied_only_between_16_byte_boundaries():
    t = torch.zeros(2, 3, 4, 48, dtype=torch.bfloat16)
    assert ops._rows16(t) [1:] == (t.data_ptr(), t.stride()) and ops._rows16(t)[0] is t
    view = t.transpose(1, 2)
    assert ops._rows16(view)[0] is view
    odd = torch.zeros(2, 3, 4, 49, dtype=torch.bfloat16)[..., 1:]
    got, ptr, strides = ops._rows16(odd)
    assert got is not odd and got.is_contiguous() and ptr == got.data_ptr() and strides == got.stride()
