"""The addresses at which the row operators' kernels take the rows of an array, compiled for the HOST and compared with
the array's strides: groups of threads step from row to row, past the end of an inner axis, over slices, reversed
axes and axes that are broadcast."""

import ctypes as C
import itertools
import os
import shutil
import subprocess

import numpy as np
import pytest

from dpnp_b200.tensor import _row_functions as rf

HERE = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(HERE, "host_harness", "row_walk_host.cu")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc is needed to build the host harness")
    out = str(tmp_path_factory.mktemp("rw") / "librw_host.so")
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "--expt-relaxed-constexpr", "-shared",
           "-Xcompiler", "-fPIC", "-x", "cu", SRC, "-o", out]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    return C.CDLL(out)


def _longs(values):
    return (C.c_int64 * max(1, len(values)))(*values)


# leading extents and strides, in elements; rows of 8
LEADING = [
    ((7,), (8,)), ((7,), (11,)), ((7,), (-8,)), ((7,), (0,)), ((), ()), ((1,), (5,)),
    ((4, 6), (0, 8)),                      # a matrix broadcast over a leading axis
    ((64, 3), (0, 8)), ((3, 64), (0, 8)), ((4, 6), (0, -8)), ((4, 6), (0, 11)),
    ((4, 6), (8, 0)), ((4, 6), (0, 0)),    # broadcast over the inner axis, over both
    ((4, 6), (100, 8)), ((4, 6), (48, 8)), ((4, 6), (-100, 8)), ((4, 6), (8, 32)), ((4, 6), (100, -9)),
    ((2, 3, 5), (0, 40, 8)), ((2, 3, 5), (200, 40, 8)), ((2, 3, 5), (0, 0, 8)), ((2, 3, 5), (8, 0, 0)),
    ((2, 1, 5), (0, 77, 8)), ((1, 4, 1, 6, 1), (9, 0, 9, 8, 9)), ((2, 3, 5), (500, 100, 8)), ((2, 3, 5), (0, 100, 8)),
    ((2, 3, 5), (40, 0, 8)),
]


@pytest.mark.parametrize("lead,strides", LEADING)
def test_rows_are_walked_where_the_strides_say(lib, lead, strides):
    shape, st = lead + (8,), strides + (1,)
    rows = int(np.prod(lead, dtype=int))
    want = [sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, lead))]
    got = (C.c_int64 * rows)()
    args = len(shape), _longs(shape), _longs(st)
    for step in (1, 2, 3, 5, 8, 16, rows, rows + 1):
        for first in range(min(step, rows)):
            n = lib.rw_walk(*args, C.c_uint32(first), C.c_uint32(step), got)
            if not rf._walkable(shape, st):
                assert n == -1
                continue
            assert n == len(want[first::step]) and list(got[:n]) == want[first::step], (first, step)


@pytest.mark.parametrize("lead,strides", LEADING)
def test_rows_count_as_one_stride_apart_only_where_they_are(lib, lead, strides):
    """(What the kernels that shift the columns of all rows alike go by.)"""
    shape, st = lead + (8,), strides + (1,)
    one = lib.rw_one_stride(len(shape), _longs(shape), _longs(st))
    if not rf._walkable(shape, st):
        assert one == -1
        return
    starts = [sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, lead))]
    assert bool(one) == (len(set(np.diff(starts))) <= 1)
