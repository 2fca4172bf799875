"""Sizes (M, N, K) for the tests of eas.ops, and the kernel each runs on."""

import ctypes

# single rows and columns, both sides of every tile edge, rows of one to several hundred
SHAPES = [(1, 1, 1), (1, 8, 8), (2, 1, 40), (3, 5, 7), (1, 4096, 1024), (4, 72, 520), (4, 2500, 72), (3, 40, 4160),
          (6, 520, 4104), (8, 300, 5000), (7, 96, 8200), (2, 1031, 96), (8, 72, 520), (9, 64, 64), (16, 200, 136),
          (17, 65, 33), (31, 8, 2088), (33, 128, 256), (64, 96, 1000), (65, 1000, 72), (128, 128, 64), (129, 257, 130),
          (200, 640, 192), (257, 255, 65), (384, 512, 128), (520, 1031, 264)]
# many tiles; of a backward pass: both products with full and partial rounds, either of them the longer
BIG = [(1024, 1536, 320), (2304, 2080, 136), (700, 4104, 512), (3000, 4200, 2600), (1000, 8200, 3000),
       (8000, 600, 2000)]
# each reaches a kernel that the ones above do not
VARIANTS = [(141, 9525, 1), (11, 2053, 2908), (5331, 1, 1863), (68, 1, 1601), (9, 10311, 1), (289, 9716, 1),
            (8, 4149, 5625), (72, 4488, 2854), (6, 2055, 7158), (2694, 66, 2214), (9, 1267, 2388), (9, 5295, 1),
            (275, 5248, 1), (4363, 37, 2853), (9, 1112, 2749), (2219, 36, 2229), (1, 1124, 2501), (3131, 1257, 1),
            (2182, 837, 1), (1755, 785, 1), (1, 1, 9666), (70, 1, 8776), (1, 1722, 4343), (3387, 1292, 72),
            (1, 1355, 2095), (1720, 1511, 66), (2247, 861, 66), (13, 2500, 1355), (1723, 515, 1),
            (2701, 1202, 51), (7, 6215, 795), (177, 7941, 170),
            (3503, 160, 408), (1, 64, 50000), (6944, 76, 3), (676, 535, 9884), (19, 9943, 2044)]

LINEAR, GATED, LINEAR_BACKWARD, GATED_BACKWARD = range(4)
DX, DW, DB = 1, 2, 4


def plan(op, m, n, k, outputs=0, sms=148):
    """(kernel, width, split of the first and second product, rows of A, CTAs per SM) of a call."""
    from easy_as_b200.runtime import cuda_ext

    v = [ctypes.c_int() for _ in range(6)]
    cuda_ext.check(cuda_ext.load().eas_dense_plan(op, m, n, k, outputs, sms, *[ctypes.byref(x) for x in v]))
    return tuple(x.value for x in v)


def kernels(shape):
    """Every way of a kernel that the exact tests run a shape on (backward passes: all outputs, and each alone): the
    kernel, its width and rows, CTAs per SM, whether the sums of each product are split, and by as many CTAs."""
    calls = [(LINEAR, 0), (GATED, 0), (LINEAR_BACKWARD, DX | DW | DB), (LINEAR_BACKWARD, DX), (LINEAR_BACKWARD, DW),
             (GATED_BACKWARD, DX | DW), (GATED_BACKWARD, DX)]
    found = set()
    for op, outputs in calls:
        kernel, width, s0, s1, rows, per_sm = plan(op, *shape, outputs)
        found.add((min(op, LINEAR_BACKWARD), kernel, width, rows, per_sm, s0 > 1, s1 > 1, s0 == s1))
    return found
