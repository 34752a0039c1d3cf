"""Sizes, addresses and waits of the MXFP4 row kernels, asked of what they are built from.  No GPU needed."""
import ctypes
import random

import pytest

from nn_amd import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("planes", [1, 3])
def test_copies_of_x_stay_in_its_planes(lib, planes):
    """The GEMM with bf16 operands copies 16 bytes at (offset of a lane) + (plane and unit, a scalar offset).  A buffer's range
    check is only sure to count the lane's offset, so that one has to keep every copy in the planes by itself: of all rows of
    the last row block, those past m too, and all columns of a unit that K ends in."""
    lib.nnq_rule_mx_x_offset.argtypes = [ctypes.c_int] * 5
    rng = random.Random(planes)
    cases = [(17, 32, 64), (33, 2880, 64), (64, 384, 64), (65, 1056, 64), (1, 160, 32), (129, 4096, 128)]
    cases += [(rng.randint(1, 300), 32 * rng.randint(1, 40), rng.choice((32, 64))) for _ in range(12)]
    for m, k, tile in cases:
        total = planes * m * k * 2
        units = (k + 127) // 128
        read = set()
        for row in range((m + tile - 1) // tile * tile):
            for u in {0, units // 2, units - 1}:
                for col in range(0, 128, 8):
                    off = lib.nnq_rule_mx_x_offset(row, m, k, u, col)
                    if off >= total:
                        assert off >= 0x7FFFFFF0 and (row >= m or 128 * u + col >= k)
                        continue
                    for plane in range(planes):
                        at = off + plane * m * k * 2 + 256 * u
                        assert at == 2 * ((plane * m + row) * k + 128 * u + col) and at + 16 <= total, (m, k, row, u, col, plane)
                    read.add((row, u, col))
        assert len(read) == m * sum(min(128, k - 128 * u) // 8 for u in {0, units // 2, units - 1})
