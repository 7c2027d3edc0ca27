"""Shapes that take each form of the group norm, and which one: a host test holds the table against the library's plan, a GPU
test holds every form to its bounds."""
import torch

SIZE = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}

# channels a group by (element, vector) bytes: a group's row piece is 48, 24, 20 or 10 bytes, so that it divides into these
GROUP = {(4, 16): 12, (4, 8): 6, (4, 4): 5, (2, 16): 24, (2, 8): 12, (2, 4): 10, (2, 2): 5}

# (B, H, W, G), registers of a thread in the forward and backward kernel that keep their slice (0: by passes), vector widths
SLICES = [((2, 9, 11, 3), 8, 8, (16, 8, 4, 2)),
          ((3, 31, 33, 7), 24, 24, (16,)),
          ((3, 49, 51, 7), 24, 24, (8, 4, 2)),
          ((2, 71, 70, 33), 64, 0, (16, 8, 4, 2)),
          ((2, 70, 71, 5), 0, 0, (16, 8, 4))]

# several groups a workgroup: (B, H, W, C, G), element bytes, groups, registers, vector bytes
CLUSTERS = [((16, 64, 64, 320, 32), 2, 2, 64, 4), ((32, 52, 52, 64, 32), 2, 4, 24, 4), ((16, 51, 51, 768, 32), 2, 2, 64, 16),
            ((16, 64, 64, 160, 32), 4, 2, 64, 4), ((32, 52, 52, 64, 32), 4, 4, 24, 8)]

# rows of 513 vectors, or more groups than threads: chunk statistics are joined by a launch of their own
JOINED = [((2, 30, 31, 513 * vb // es, 3), es, vb) for es in (4, 2) for vb in (16, 8, 4, 2) if vb >= es]


def vectors(regs, vb):
    return regs * 4 // vb if vb >= 4 else regs


def cases():
    """(B, H, W, C, G), dtype, expected plan of both directions: vectors a thread, vector bytes, groups, joined by passes."""
    for dtype, es in SIZE.items():
        for (B, H, W, G), fwd, bwd, widths in SLICES:
            for vb in widths:
                if (es, vb) in GROUP:
                    C = GROUP[es, vb] * G
                    yield (B, H, W, C, G), dtype, (vectors(fwd, vb), vb if fwd else None, 1, 1), (vectors(bwd, vb), vb if bwd else None, 1, 1)
        for shape, size, gc, regs, vb in CLUSTERS:
            if size == es:
                yield shape, dtype, (vectors(regs, vb), vb, gc, 1), None
        for shape, size, vb in JOINED:
            if size == es:
                yield shape, dtype, (0, vb, 1, 0), (0, vb, 1, 0)
    yield (1, 100, 83, 1200, 600), torch.float32, None, (0, 16, 1, 0)


CASES = list(cases())
IDS = ["%s %s" % ("x".join(map(str, s)), str(t)[6:]) for s, t, _, _ in CASES]
