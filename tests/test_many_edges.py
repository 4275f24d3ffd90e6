"""Scratch of attention of several queries: found on the host, nothing is launched."""
import ctypes

import pytest


@pytest.mark.parametrize("D,dtype,queries,tokens", [(128, 2, 512, 4096), (64, 1, 300, 9000), (96, 0, 100, 2000), (256, 2, 2048, 40000)])
def test_scratch_is_what_launches_use(pkg, D, dtype, queries, tokens):
    """Rows that are in one split are finished in the block that has them: no scratch, however many queries there are.  Sums of what keys receive need the queries' operands
    (two fp16 terms of every coordinate), 64 statistics and a scale a tile of 32 at least; kernels for all dimensions need the operands in any case."""
    native = pkg._native
    r = native.TqAttendRequest(batch=8, heads=8, group=4, n_queries=queries, tokens=tokens, head_dim=D, dtype=dtype, bits_k=4, bits_v=4, scale=1.0)
    r.window.tokens = 128
    scratch = lambda: native.lib().tq_attend_many_scratch(ctypes.byref(r))  # noqa: E731
    tiles = 64 * -(-4 * queries // 32)
    assert scratch() == 4
    r.weights = 4096
    assert scratch() >= tiles * (32 * D + 64 + 1)
    r.weights, r.tokens = None, 31
    assert scratch() >= tiles * 32 * D
