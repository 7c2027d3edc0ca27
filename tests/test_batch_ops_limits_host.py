"""The largest sizes that the 8-bit cache, shared-prefix attention and group norm take: what their index arithmetic or a launch
cannot hold is refused on the host, before any GPU call."""
import pytest

from style_transfer_amd import lib

A = 1 << 20                 # an aligned address that nothing reads


def norm(B, N, C, G, dtype=lib.DTYPE_BF16, backward=False, ws_bytes=0):
    """No workspace: what passes the size checks and takes the passes ends with -12, before a launch."""
    L = lib.load()
    if backward:
        rc = L.sid_group_norm_act_bwd(A, A, A, A, A, A, A, A, A, B, N, C, G, 1, dtype, A, ws_bytes, None)
    else:
        rc = L.sid_group_norm_act_fwd(A, A, A, A, A, A, B, N, C, G, 1e-5, 1, dtype, A, ws_bytes, None)
    return rc, L.sid_last_error().decode()


@pytest.mark.parametrize("N", [2 ** 31 - 1, 2 ** 31 - 4096, 2 ** 31 - 2 ** 16])
def test_group_norm_rows_near_31_bits(N):
    """A pass walks rows in 32-bit integers, up to eight rows of 512 threads and one chunk's rounding ahead of the last row:
    within 2^16 of 2^31 the row behind the end would be negative, and read."""
    L = lib.load()
    assert L.sid_group_norm_workspace_bytes(1, N, 1, 1, lib.DTYPE_BF16, 0) == 0 and "too large" in L.sid_last_error().decode()
    for backward in (False, True):
        rc, msg = norm(1, N, 1, 1, backward=backward)
        assert rc == -22 and "too large" in msg
    # the largest that is taken: refused here for its workspace alone
    assert L.sid_group_norm_workspace_bytes(1, 2 ** 31 - 2 ** 16 - 1, 1, 1, lib.DTYPE_BF16, 0) > 256
    assert norm(1, 2 ** 31 - 2 ** 16 - 1, 1, 1)[0] == norm(1, 2 ** 31 - 2 ** 16 - 1, 1, 1, backward=True)[0] == -12


def test_group_norm_backward_takes_any_gradient_alone():
    """No dx: refused for its workspace alone here, as with it.  None of the three: nothing to do."""
    L = lib.load()
    call = lambda dx, dw, db: L.sid_group_norm_act_bwd(A, A, A, A, A, A, dx, dw, db, 1, 1 << 16, 64, 8, 1, lib.DTYPE_F32, A, 0, None)
    assert call(A, A, A) == call(None, A, A) == call(None, None, A) == call(None, A, None) == call(A, None, None) == -12
    assert call(None, None, None) == -22 and "no gradient" in L.sid_last_error().decode()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("B,N,C,G", [(65535, 1, 512, 512),        # one workgroup a group: 2^25 of them
                                     (1, 1, 1 << 28, 1),          # 2^16 slabs of 512 vectors
                                     (1, 1, (1 << 27) - 31, 1)])  # 32 threads a channel
def test_group_norm_beyond_one_launch(B, N, C, G, backward):
    rc, msg = norm(B, N, C, G, backward=backward)
    assert rc == -22 and "too large" in msg, (rc, msg)


def test_cache_write_beyond_one_launch():
    """2^24 workgroups of eight rows."""
    L, s = lib.load(), lib.strides3(256, 256, 256)
    rc = L.sid_kv_cache_write(A, A, s, s, A, A, A, A, A, None, 1, 1, 1 << 27, 1, 256, lib.DTYPE_BF16, lib.KV_INT8, None)
    assert rc == -22 and "too many rows" in L.sid_last_error().decode()


def test_shared_attention_beyond_one_launch():
    """2^24 workgroups: as many sequences of one query, each with keys of its own."""
    L, q = lib.load(), lib.strides3(8, 8, 8)
    src = lib.kv_source(A, A, 0, 0, 8, 8, 8, 8, 8, 8, 0, 0, lib.KV_NONE)
    rc = L.sid_shared_attn_fwd(A, q, src, src, None, A, (1 << 24) - 1, 1, 1, 1, 8, 8, 8, 1.0, 0, lib.DTYPE_BF16, A, 0, None)
    assert rc == -22 and "too many rows" in L.sid_last_error().decode()
