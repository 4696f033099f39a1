"""The index arithmetic of the paged KV cache, on the CPU: the header the
kernels use, compiled for the host.  Whatever the lengths, bounds and rows say,
a position that counts as good lies in what the table names, rows of the pool
are a bijection of (page, head, offset), and the attention's chunks cover each
sequence once, no more of them than the grid and the partials have room for."""
import ctypes
import itertools
import os
import random
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
    U32, I32 = ctypes.c_uint32, ctypes.c_int32
    L.quotient.argtypes, L.quotient.restype = [U32] * 2, U32
    L.limit_of.argtypes, L.limit_of.restype = [I64] * 4, I64
    L.count_of.argtypes = [I32, I64]
    L.chunk_len_of.argtypes = [I32] * 3
    L.cut_of.argtypes = [I64] * 3 + [ctypes.POINTER(I64)]
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


def test_quotients(lib):
    rng = random.Random(1)
    for d in [1, 2, 3, 5, 7, 15, 16, 17, 24, 48, 64, 640, 641, 65535, 65536, 2**30 - 1, 2**30, 2**30 + 1, I32_MAX] + \
            [rng.randrange(1, I32_MAX) for _ in range(200)]:
        ns = [0, 1, d - 1, d, 2 * d - 1, I32_MAX - 1, I32_MAX] + [rng.randrange(I32_MAX) for _ in range(20)]
        ns += [k * d + e for k in (1, 2, I32_MAX // d) for e in (-1, 0, 1)]
        for n in ns:
            if 0 <= n <= I32_MAX:
                assert lib.quotient(n, d) == n // d, (n, d)


@pytest.mark.parametrize("unit", [64, 128])
def test_chunks_cover_each_sequence_within_bounds(lib, unit):
    rng = random.Random(2)
    cases = [[1], [0], [0] * 70, [64], [65], [I32_MAX], [I32_MAX] * 5, [100000] + [1] * 63, [1] * 3000]
    for _ in range(300):
        hi = 10 ** rng.randint(0, 9)
        cases.append([rng.randint(0, hi) for _ in range(rng.randint(1, 80))])
    for lens in cases:
        for target in (1, 7, 128, 1024):
            least = -(-max(lens) // 2048)
            limit = lib.limit_of(sum(lens), target, least, unit)
            assert limit % unit == 0 and limit >= unit and limit >= least
            chunks = slots = 0
            for n in lens:
                c = lib.count_of(n, limit)
                size = lib.chunk_len_of(n, c, unit)
                assert c >= 1 and (c - 1) * limit <= n <= c * limit
                assert c * size >= n and (c == 1 or (size % unit == 0 and size <= limit))
                assert c <= max(1, -(-n // unit)) and c <= 2048
                chunks += c
                slots += c if c > 1 else 0
            assert chunks <= target + 1 + len(lens)
            assert slots <= 2 * target + 2


@pytest.mark.parametrize("seqs", [1, 2, 7, 63, 64, 65, 256, 257, 1000, 5000])
@pytest.mark.parametrize("parts", [1, 3, 8, 16, 600])
def test_chunks_fit_the_launch(lib, seqs, parts):
    """For any lengths up to the table's positions: no more chunks than blocks,
    no more chunks of cut sequences than partials, of one sequence than its
    join holds; none cut where no join is launched."""
    rng = random.Random(seqs * 31 + parts)
    shape = (ctypes.c_int64 * 6)()
    for cap in (0, 1, 511, 512, 513, 1024, 1025, 4096, 100_001, 3_000_000, I32_MAX):
        cut = lib.cut_of(seqs, cap, parts, shape)
        target, least, room, slots, most, unit = shape
        for kind in range(6):
            lens = {0: lambda: cap, 1: lambda: 0, 2: lambda: rng.randint(0, cap), 3: lambda: min(cap, 513),
                    4: lambda: min(cap, rng.choice((0, 1, unit, unit + 1, 1100))),
                    5: lambda: cap if rng.random() < 2 / seqs else min(cap, 3)}[kind]
            lens = [lens() for _ in range(seqs)]
            limit = lib.limit_of(sum(lens), target, least, unit)
            counts = [lib.count_of(n, limit) for n in lens]
            assert sum(counts) <= room
            assert max(counts) <= (min(most, max(slots, 1)) if cut else 1)
            assert sum(c for c in counts if c > 1) <= slots
            assert all(lib.chunk_len_of(n, c, unit) * c >= n for n, c in zip(lens, counts))
