"""Which form of the group norm a shape takes: a threshold that moves must not leave a form without its test."""
import ctypes

import pytest
import torch

from group_norm_forms import CASES, IDS
from style_transfer_amd import lib

CODE = {torch.float32: lib.DTYPE_F32, torch.bfloat16: lib.DTYPE_BF16, torch.float16: lib.DTYPE_F16}


def plan(shape, dtype, backward):
    B, H, W, C, G = shape
    p = (ctypes.c_int * 6)()
    lib.check(lib.load().sid_group_norm_plan(B, H * W, C, G, CODE[dtype], int(backward), p))
    return list(p)


@pytest.mark.parametrize("shape,dtype,fwd,bwd", CASES, ids=IDS)
def test_shape_takes_its_form(shape, dtype, fwd, bwd):
    for backward, want in ((False, fwd), (True, bwd)):
        if want is None:
            continue
        nv, vb, threads, gc, chunks, fold = plan(shape, dtype, backward)
        assert (nv, gc) == (want[0], want[2]) and want[1] in (None, vb)
        assert 256 <= threads <= 1024 and (chunks >= 1) == (nv == 0)
        if nv == 0:
            assert fold == want[3]


def test_every_kept_slice_has_a_shape():
    """Each (type, vector width, registers) of the two kernels that keep their slice, and 2 and 4 groups a workgroup."""
    have = [set(), set()]
    groups = set()
    for shape, dtype, _, _ in CASES:
        for backward in (False, True):
            nv, vb, _, gc, _, _ = plan(shape, dtype, backward)
            if nv:
                have[backward].add((dtype, vb, nv))
                groups.add(gc)
    for backward, classes in ((False, (8, 24, 64)), (True, (8, 24))):
        for dtype, widths in ((torch.float32, (16, 8, 4)), (torch.bfloat16, (16, 8, 4, 2)), (torch.float16, (16, 8, 4, 2))):
            for vb in widths:
                for regs in classes:
                    assert (dtype, vb, regs * 4 // vb if vb >= 4 else regs) in have[backward], (backward, dtype, vb, regs)
    assert groups == {1, 2, 4}


def test_plan_refusals():
    L, p = lib.load(), (ctypes.c_int * 6)()
    assert L.sid_group_norm_plan(1, 4, 64, 7, 0, 0, p) == -22 and L.sid_group_norm_plan(1, 4, 64, 8, 0, 0, None) == -22
