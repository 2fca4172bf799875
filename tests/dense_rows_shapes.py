"""Sizes (M, N, K) of up to 8 rows for the tests of eas.ops, and the way that each runs on."""

import ctypes

#: run with rows on 16 bytes (where K lets them be) and at odd addresses
SHAPES = [(1, 1, 1), (2, 40, 72), (3, 7, 1030), (1, 2100, 1025), (8, 33, 130), (1, 700, 4104), (2, 300, 8200), (5, 264, 5000),
          (8, 520, 4099), (3, 600, 8203), (3, 520, 8203), (2, 520, 16390), (4, 1500, 8195), (7, 1400, 5003), (2, 5000, 520),
          (8, 4300, 5001), (1, 520, 4200), (1, 1180, 20001), (1, 70, 40001), (3, 37, 9001)]

WORDS, SHIFTED, VALUES = range(3)


def plan(gated, m, n, k, unaligned, sms=148):
    """(way of reading the weights, warps per block, CTAs that share K)"""
    from easy_as_b200.runtime import cuda_ext

    v = [ctypes.c_int() for _ in range(3)]
    cuda_ext.check(cuda_ext.load().eas_dense_rows_plan(int(gated), m, n, k, 7 if unaligned else 0, sms,
                                                       *[ctypes.byref(x) for x in v]))
    return tuple(x.value for x in v)


def ways(shape):
    m, _n, k = shape
    return {(gated, *plan(gated, *shape, odd)) for gated in (False, True) for odd in (False, True)}
