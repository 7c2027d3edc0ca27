"""Every form of the group norm -- each register class and vector width, several groups a workgroup, passes with either join --
forward and gradients against 64 bits, at the bounds of test_gpu_group_norm.py (whose longest chain of additions, 200, holds
here too: 128 of a thread's 64 registers of 16-bit values, 6 of a wave, 16 of the workgroup; 117 chunks in a row behind 8 rows
of a thread)."""
import pytest

import test_gpu_group_norm as base
from group_norm_forms import CASES, IDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,dtype", [c[:2] for c in CASES], ids=IDS)
def test_form(shape, dtype):
    base.test_forward_and_gradients(*shape, dtype, "silu")


@pytest.mark.parametrize("shape,dtype", [c[:2] for c in CASES if c[2] and c[2][2] > 1])
def test_groups_of_one_workgroup_keep_apart(shape, dtype):
    """Groups whose means and spreads differ by their number: one's statistics would show in another's values."""
    import torch
    B, H, W, C, G = shape
    o = base.ops()
    x, w, b, _ = base.make(B, H, W, C, dtype, 3)
    g = torch.arange(C, device="cuda") // (C // G)
    x = (x.float() * (1 + g % 4).view(1, -1, 1, 1) + (g % 4).view(1, -1, 1, 1)).to(dtype).contiguous(memory_format=torch.channels_last)
    got = o.group_norm_act(x, G, w, b, act="none")
    Y, xh, stat = base.oracle(x, w, b, G, 1e-5, "none")
    bound = (base.xh_error(xh, stat, x, G) + 4 * base.F32 * (xh.abs() + 1)) * w.double().abs().view(1, -1, 1, 1) + 4 * base.F32 * Y.abs()
    assert bool(((got.double() - Y).abs() <= bound + base.HALF[dtype] * Y.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)).all())
