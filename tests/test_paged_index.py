"""The index arithmetic of the paged KV cache, on the CPU: the header the
kernels use, compiled for the host.  Whatever the lengths, bounds and rows say,
a position that counts as good lies in what the table names, and rows of the
pool are a bijection of (page, head, offset)."""
import ctypes
import itertools
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OK, IDLE, BAD = 0, 1, 2
I32_MIN, I32_MAX = -2**31, 2**31 - 1


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("paged") / "libpaged_index.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                    os.path.join(HERE, "paged_index.cpp"), "-o", str(so)], check=True)
    L = ctypes.CDLL(str(so))
    I64 = ctypes.c_int64
    L.pos_of.argtypes = [I64] * 5 + [ctypes.POINTER(I64)]
    L.row_of.argtypes, L.row_of.restype = [I64] * 5, I64
    L.len_of.argtypes, L.len_of.restype = [I64] * 2, I64
    return L


def pos_of(lib, *a):
    p = ctypes.c_int64()
    return lib.pos_of(*a, ctypes.byref(p)), p.value


def test_new_rows_take_the_last_positions(lib):
    for new, old in itertools.product((1, 2, 5), (0, 1, 7)):
        got = [pos_of(lib, 10 + i, 10, 10 + new, old + new, 64) for i in range(new)]
        assert got == [(OK, old + i) for i in range(new)]


def test_a_length_of_zero_is_idle(lib):
    assert pos_of(lib, 3, 3, 4, 0, 64)[0] == IDLE


@pytest.mark.parametrize("r,first,end,length,cap", [
    (5, 4, 8, 3, 64),            # more new rows than the length
    (5, 4, 6, 65, 64),           # a length beyond the table's positions
    (5, 4, 6, -1, 64),
    (5, 4, 6, I32_MIN, 64),
    (5, 4, 6, I32_MAX, 64),
    (3, 4, 6, 9, 64),            # rows before the first bound
    (6, 4, 6, 9, 64),
    (5, 6, 4, 9, 64),            # bounds that descend
    (5, I32_MIN, I32_MAX, 9, 64),
])
def test_bad_rows(lib, r, first, end, length, cap):
    assert pos_of(lib, r, first, end, length, cap)[0] == BAD


def test_good_positions_lie_in_the_table(lib):
    edge = (I32_MIN, -1, 0, 1, 2, 15, 16, 17, I32_MAX)
    for r, first, end, length in itertools.product((0, 1, 16), edge, edge, edge):
        state, pos = pos_of(lib, r, first, end, length, 16)
        if state == OK:
            assert 0 <= pos < 16 and pos < length
        assert lib.len_of(length, 16) == (length if 0 <= length <= 16 else 0)


def test_pool_rows_are_a_bijection(lib):
    pages, kv, page = 3, 2, 5
    rows = [lib.row_of(p, j, o, kv, page) for p in range(pages) for j in range(kv) for o in range(page)]
    assert rows == list(range(pages * kv * page))
    # Past 32 bits.
    assert lib.row_of(1 << 20, 7, 63, 8, 64) == ((1 << 20) * 8 + 7) * 64 + 63
