"""The paged KV cache on the device: mi_qkv_rope_paged and mi_paged_attention.

The append against numpy: RoPE's two products and one sum, each rounded, bit
for bit, BF16 stores rounded to nearest even; every slot of the pools that no
new position names stays as it was, bit for bit.

The attention against float64, F32 or BF16 pools.  Its tolerance per output
value, with u = 2^-24: a score is a sum of D products, so it is off by at most
(D + 2) u A, A the largest scale * sum |q k| over the positions, and its
difference to the maximum by twice that and a rounding; e^x passes that on as a
relative error of the weight (with 4 u of its own), the sums of up to n
weights and of n weighted values add n u each, the join and the division a few
more: u (4 (D + 8) A + 2 n + 64) sum p |v| (BF16 results: 2^-8 of the value
besides).

Slots outside the sequences' positions hold NaN and table entries behind a
sequence's last page are out of range, so a read of either is seen.
"""
import threading

import numpy as np
import pytest

import miburn
from miburn import BF16, F32

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.fixture(scope="module")
def eng():
    e = miburn.Engine(0)
    yield e
    e.close()


def bits(x):
    return np.ascontiguousarray(x).view({2: np.uint16, 4: np.uint32}[x.dtype.itemsize])


def put(eng, x, elem):
    """F32 values in a buffer of `elem`, and as the buffer holds them."""
    x = np.ascontiguousarray(x, np.float32)
    if elem == F32:
        return eng.upload(x), x
    b = miburn.bf16_bits(x)
    return eng.upload_bf16(b.reshape(x.shape)), miburn.bf16_to_f32(b).reshape(x.shape)


def get(eng, id_):
    y = eng.download(id_)
    return miburn.bf16_to_f32(y).reshape(y.shape) if y.dtype == np.uint16 else y


class Cache:
    """A pool of shuffled pages with one table row a sequence."""

    def __init__(self, rng, lens, kv, d, page, elem, spare=2, width=None):
        self.lens, self.kv, self.d, self.page, self.elem = list(lens), kv, d, page, elem
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        width = width or max(1, max(need, default=1))
        # Behind a sequence's last page: values that name no page.
        self.table = np.where(rng.random((len(lens), width)) < 0.5, -1, 2**31 - 1).astype(np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        rows = self.pages * kv * page
        self.k = rng.standard_normal((rows, d)).astype(np.float32)
        self.v = rng.standard_normal((rows, d)).astype(np.float32)
        if elem == BF16:
            self.k, self.v = (miburn.bf16_to_f32(miburn.bf16_bits(x)).reshape(rows, d) for x in (self.k, self.v))

    def row(self, s, pos, j):
        return (int(self.table[s, pos // self.page]) * self.kv + j) * self.page + pos % self.page

    def rows(self, s, j):
        pos = np.arange(self.lens[s])
        return (self.table[s, pos // self.page].astype(np.int64) * self.kv + j) * self.page + pos % self.page

    def poison(self):
        """NaN in every slot that no sequence's positions name."""
        used = np.zeros(self.k.shape[0], bool)
        for s in range(len(self.lens)):
            for j in range(self.kv):
                used[self.rows(s, j)] = True
        self.k[~used] = np.nan
        self.v[~used] = np.nan
        return self

    def up(self, eng):
        self.kid, self.vid = put(eng, self.k, self.elem)[0], put(eng, self.v, self.elem)[0]
        self.tid = eng.upload_i32(self.table)
        self.lid = eng.upload_i32(np.array(self.lens, np.int32).reshape(-1, 1))
        return self


def rope_tables(n, d, theta=1e5):
    ang = np.arange(n)[:, None] * (theta ** (-np.arange(0, d, 2, dtype=np.float64) / d))[None, :]
    return (np.concatenate([np.cos(ang), np.cos(ang)], 1).astype(np.float32),
            np.concatenate([-np.sin(ang), np.sin(ang)], 1).astype(np.float32))


def rope(x, cos, sin):
    """x [heads, d] F32 at one position's table rows."""
    half = x.shape[-1] // 2
    return x * cos + np.concatenate([x[..., half:], x[..., :half]], -1) * sin


# ------------------------------------------------------------------ append


def append_case(eng, rng, lens, news, heads, kv, d, page, xe, ce, oe, starts=True, extra=0, spare=2):
    c = Cache(rng, lens, kv, d, page, ce, spare).up(eng)
    rows = sum(news) + extra
    xid, x = put(eng, rng.standard_normal((rows, (heads + 2 * kv) * d)), xe)
    cos, sin = rope_tables(max(max(lens), 1), d)
    cid, sid = eng.upload(cos), eng.upload(sin)
    bounds = np.concatenate([[0], np.cumsum(news)]).astype(np.int32).reshape(-1, 1)
    stid = eng.upload_i32(bounds) if starts else 0
    qid = eng.qkv_rope_paged(xid, cid, sid, c.tid, c.lid, stid, heads, kv, page, c.kid, c.vid, oe)
    want_k, want_v = c.k.copy(), c.v.copy()
    want_q = np.zeros((rows, heads, d), np.float32)
    r = 0
    for s, n in enumerate(news):
        for i in range(n):
            if lens[s] > 0:
                pos = lens[s] - n + i
                h = x[r].reshape(-1, d)
                want_q[r] = rope(h[:heads], cos[pos], sin[pos])
                k = rope(h[heads:heads + kv], cos[pos], sin[pos])
                for j in range(kv):
                    want_k[c.row(s, pos, j)] = k[j]
                    want_v[c.row(s, pos, j)] = h[heads + kv + j]
            r += 1
    return c, qid, want_q.reshape(rows, heads * d), want_k, want_v


def same(eng, id_, want, elem):
    got = eng.download(id_)
    want = np.ascontiguousarray(want, np.float32)
    w = miburn.bf16_bits(want).reshape(want.shape) if elem == BF16 else want
    bad = np.flatnonzero(bits(got) != bits(w))
    assert bad.size == 0, f"{bad.size} datums differ, first at {bad[0]} of {got.shape}"


@pytest.mark.parametrize("xe,ce,oe", [(F32, F32, F32), (F32, BF16, F32), (BF16, BF16, BF16), (BF16, F32, F32),
                                      (F32, F32, BF16)])
@pytest.mark.parametrize("lens,news,heads,kv,d,page", [
    ([1], [1], 1, 1, 16, 1),
    ([577], [1], 9, 3, 64, 16),
    ([1, 16, 17, 0, 33, 100], [1] * 6, 4, 2, 32, 16),
    ([5, 12, 0, 40], [5, 1, 0, 37], 6, 2, 64, 8),
    ([31, 7, 300], [30, 7, 129], 8, 1, 128, 48),
    ([129], [129], 3, 3, 16, 640),
])
def test_append_bits(eng, lens, news, heads, kv, d, page, xe, ce, oe):
    rng = np.random.default_rng(11 + d + page)
    starts = any(n != 1 for n in news)
    c, qid, q, k, v = append_case(eng, rng, lens, news, heads, kv, d, page, xe, ce, oe, starts)
    same(eng, qid, q, oe)
    same(eng, c.kid, k, ce)
    same(eng, c.vid, v, ce)
    eng.sync()


def test_append_many_sequences(eng):
    """More sequences than a wavefront's lanes, some with no rows."""
    rng = np.random.default_rng(3)
    news = [int(n) for n in rng.integers(0, 4, 200)]
    lens = [n + int(e) if n else int(e) for n, e in zip(news, rng.integers(0, 40, 200))]
    c, qid, q, k, v = append_case(eng, rng, lens, news, 4, 2, 32, 16, F32, BF16, F32)
    same(eng, qid, q, F32)
    same(eng, c.kid, k, BF16)
    same(eng, c.vid, v, BF16)
    eng.sync()


def test_append_padded_batch(eng):
    """Idle sequences and rows behind the last sequence write nothing and
    give zeros."""
    rng = np.random.default_rng(5)
    c, qid, q, k, v = append_case(eng, rng, [4, 0, 9], [2, 3, 4], 4, 2, 64, 16, F32, F32, F32, extra=6)
    same(eng, qid, q, F32)
    assert not q[2:5].any() and not q[9:].any()
    same(eng, c.kid, k, F32)
    same(eng, c.vid, v, F32)
    eng.sync()


def test_append_into_one_slot_equals_the_contiguous_cache(eng):
    """A cache of one slot a sequence is one of pages of max_ctx: the same
    bits as mi_qkv_rope_cache."""
    rng = np.random.default_rng(6)
    batch, seq, pos0, heads, kv, d, maxc = 3, 7, 5, 6, 2, 64, 20
    x = eng.upload(rng.standard_normal((batch * seq, (heads + 2 * kv) * d)))
    cos, sin = (eng.upload(t) for t in rope_tables(maxc, d))
    pools = [eng.upload(np.zeros((batch * kv * maxc, d), np.float32)) for _ in range(4)]
    q0 = eng.qkv_rope_cache(x, cos, sin, seq, heads, kv, pos0, pools[0], pools[1])
    table = eng.upload_i32(np.arange(batch).reshape(-1, 1))
    lens = eng.upload_i32(np.full((batch, 1), pos0 + seq))
    starts = eng.upload_i32(np.arange(batch + 1).reshape(-1, 1) * seq)
    q1 = eng.qkv_rope_paged(x, cos, sin, table, lens, starts, heads, kv, maxc, pools[2], pools[3])
    assert eng.metadata(q1) == (batch * seq, heads * d, F32)
    assert np.array_equal(bits(eng.download(q0)).ravel(), bits(eng.download(q1)).ravel())
    for a, b in ((0, 2), (1, 3)):
        assert np.array_equal(bits(eng.download(pools[a])), bits(eng.download(pools[b])))


@pytest.mark.parametrize("spoil", ["page", "page_high", "long", "short", "starts", "tables"])
def test_append_out_of_range(eng, spoil):
    """A row that names no slot writes nothing, gives zeros and is reported at
    the next wait; its neighbours are written."""
    rng = np.random.default_rng(8)
    lens, heads, kv, d, page = [9, 20, 3], 4, 2, 32, 8
    c = Cache(rng, lens, kv, d, page, F32, width=3)
    bad = 1
    starts = np.arange(4, dtype=np.int32)
    positions = 24
    if spoil == "page":
        c.table[1, 2] = -5
    elif spoil == "page_high":
        c.table[1, 2] = c.pages
    elif spoil == "long":
        c.lens[1] = 25
    elif spoil == "short":
        c.lens[1] = -3
    elif spoil == "starts":
        starts[:] = [0, 3, 2, 3]  # descending: rows 0 .. 2 of no good bounds
    else:
        positions = 19
    c.up(eng)
    x = rng.standard_normal((3, (heads + 2 * kv) * d)).astype(np.float32)
    cos, sin = rope_tables(positions, d)
    qid = eng.qkv_rope_paged(eng.upload(x), eng.upload(cos), eng.upload(sin), c.tid, c.lid,
                             eng.upload_i32(starts.reshape(-1, 1)) if spoil == "starts" else 0, heads, kv, page,
                             c.kid, c.vid)
    with pytest.raises(miburn.MiError) as e:
        eng.sync()
    assert e.value.kind == "DOMAIN"
    if spoil == "starts":
        return
    q = eng.download(qid).reshape(3, heads, d)
    k, v = c.k.copy(), c.v.copy()
    for s in (0, 2):
        pos = lens[s] - 1
        h = x[s].reshape(-1, d)
        assert np.array_equal(bits(q[s]), bits(rope(h[:heads], cos[pos], sin[pos])))
        for j in range(kv):
            k[c.row(s, pos, j)], v[c.row(s, pos, j)] = rope(h[heads + j], cos[pos], sin[pos]), h[heads + kv + j]
    assert not q[bad].any()
    same(eng, c.kid, k, F32)
    same(eng, c.vid, v, F32)


# --------------------------------------------------------------- attention


def attend64(c, q, heads, scale):
    """(result, tolerance) per value, in float64."""
    S, d = len(c.lens), c.d
    q = q.reshape(S, heads, d).astype(np.float64)
    out, tol = np.zeros((S, heads, d)), np.zeros((S, heads, d))
    for s, n in enumerate(c.lens):
        if n == 0:
            continue
        for h in range(heads):
            rows = c.rows(s, h // (heads // c.kv))
            k, v = c.k[rows].astype(np.float64), c.v[rows].astype(np.float64)
            x = k @ q[s, h] * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            A = (np.abs(k) @ np.abs(q[s, h]) * abs(scale)).max()
            out[s, h] = p @ v
            tol[s, h] = U * (4 * (d + 8) * A + 2 * n + 64) * (p @ np.abs(v))
    return out.reshape(S, heads * d), tol.reshape(S, heads * d)


def attend_check(eng, c, heads, qe=F32, oe=F32, seed=1, scale=None):
    rng = np.random.default_rng(seed)
    scale = float(np.float32(c.d ** -0.5)) if scale is None else scale
    qid, q = put(eng, rng.standard_normal((len(c.lens), heads * c.d)), qe)
    oid = eng.paged_attention(qid, c.kid, c.vid, c.tid, c.lid, heads, c.kv, c.page, scale, oe)
    assert eng.metadata(oid) == (len(c.lens), heads * c.d, oe)
    got = get(eng, oid).astype(np.float64)
    want, tol = attend64(c, q, heads, scale)
    tol = tol + (2.0**-8 * np.abs(want) if oe == BF16 else 0)
    off = np.abs(got - want)
    assert np.all(off <= tol), f"worst {np.nanmax(off / np.maximum(tol, 1e-300))} of the tolerance, " \
                               f"{np.isnan(got).sum()} NaN, at {np.argwhere(~(off <= tol))[0]}"
    eng.sync()
    return qid, oid


@pytest.mark.parametrize("ce", [F32, BF16])
@pytest.mark.parametrize("heads,kv,d,page", [(9, 3, 64, 16), (1, 1, 16, 1), (4, 2, 32, 8), (8, 1, 128, 48),
                                             (12, 1, 128, 64), (16, 4, 64, 7), (5, 5, 32, 16), (40, 8, 128, 16),
                                             (20, 1, 16, 5), (64, 2, 64, 33)])
def test_attention_lengths(eng, heads, kv, d, page, ce):
    """Lengths around pages, wavefronts and tiles, and idle sequences."""
    rng = np.random.default_rng(heads * 100 + d)
    lens = [1, 0, page, page + 1, max(1, page - 1), 15, 16, 17, 31, 33, 63, 64, 65, 0, 127, 129, 200, 333]
    attend_check(eng, Cache(rng, lens, kv, d, page, ce).poison().up(eng), heads)


@pytest.mark.parametrize("qe", [F32, BF16])
@pytest.mark.parametrize("oe", [F32, BF16])
@pytest.mark.parametrize("ce", [F32, BF16])
def test_attention_types(eng, qe, ce, oe):
    rng = np.random.default_rng(4)
    for heads, kv, d in ((9, 3, 64), (8, 2, 128), (4, 4, 32), (6, 2, 16)):
        attend_check(eng, Cache(rng, [700, 1, 0, 90], kv, d, 16, ce).poison().up(eng), heads, qe, oe)


@pytest.mark.parametrize("ce", [F32, BF16])
@pytest.mark.parametrize("lens,heads,kv,d,page", [
    ([1], 9, 3, 64, 16), ([577], 9, 3, 64, 16), ([20011], 8, 2, 64, 64), ([9001, 3, 0, 4097], 24, 2, 128, 48),
    ([6000], 4, 4, 32, 6000), ([1] * 300, 4, 1, 16, 16),
    ([5000] + list(range(200)), 6, 2, 64, 16),
    (list(range(70)) + [3000, 0, 2500], 4, 2, 16, 8),
    ([int(17 * i % 90) for i in range(2500)], 2, 1, 16, 16),
])
def test_attention_splits(eng, lens, heads, kv, d, page, ce):
    """One long sequence, one long among short ones, more sequences than a
    wavefront has lanes, many short ones."""
    rng = np.random.default_rng(len(lens) + d)
    attend_check(eng, Cache(rng, lens, kv, d, page, ce).poison().up(eng), heads)


@pytest.mark.parametrize("ce", [F32, BF16])
@pytest.mark.parametrize("seqs,most,heads,kv,d,page", [
    (63, 700, 4, 2, 32, 16), (64, 1100, 2, 1, 64, 16), (65, 700, 6, 2, 16, 8), (128, 513, 4, 4, 16, 16),
    (255, 1030, 4, 1, 32, 48), (256, 600, 2, 2, 64, 16), (257, 600, 3, 1, 128, 16), (1024, 520, 2, 1, 16, 8),
    (1025, 1100, 2, 1, 16, 16), (40, 512, 4, 2, 32, 16), (40, 528, 2, 1, 32, 16), (70, 1024, 4, 2, 32, 16),
])
def test_attention_of_cuts_around_their_bounds(eng, seqs, most, heads, kv, d, page, ce):
    """Sequence counts and table widths on both sides of where the cut of the
    sequences is formed in another way or left out; empty ones in between."""
    rng = np.random.default_rng(seqs + most)
    lens = [int(n) if n % 7 else 0 for n in rng.integers(0, most // 3, seqs)]
    for at in {0, 1, 3, 4, seqs // 2, seqs - 2, seqs - 1}:
        lens[at] = most - at % 3
    attend_check(eng, Cache(rng, lens, kv, d, page, ce).poison().up(eng), heads)


@pytest.mark.parametrize("seqs", [64, 200, 300])
@pytest.mark.parametrize("live", [0, 1, 2])
def test_attention_of_few_live_sequences_among_many(eng, seqs, live):
    """All chunks are one sequence's; the idle ones' results are zeros."""
    rng = np.random.default_rng(seqs + live)
    lens = [0] * seqs
    for i in range(live):
        lens[seqs - 1 - 33 * i] = 2600 - i
    attend_check(eng, Cache(rng, lens, 2, 32, 16, BF16, width=200).poison().up(eng), 4)


@pytest.mark.parametrize("seqs", [70, 300])
def test_attention_reports_one_bad_length_among_many(eng, seqs):
    """A length out of range in a lane's second place, and one that only the
    plan's own launch sees."""
    rng = np.random.default_rng(seqs)
    c = Cache(rng, [600] * 2 + [5] * (seqs - 2), 1, 16, 16, F32)
    c.lens[seqs - 3] = -1
    c.up(eng)
    q = eng.upload(rng.standard_normal((seqs, 32)))
    out = eng.paged_attention(q, c.kid, c.vid, c.tid, c.lid, 2, 1, 16, 0.25)
    with pytest.raises(miburn.MiError) as e:
        eng.sync()
    assert e.value.kind == "DOMAIN"
    assert not eng.download(out)[seqs - 3].any()
    eng.sync()


def test_attention_no_live_sequence(eng):
    rng = np.random.default_rng(9)
    c = Cache(rng, [0, 0, 0], 2, 64, 16, BF16).poison().up(eng)
    _, oid = attend_check(eng, c, 4)
    assert not eng.download(oid).any()


def test_attention_of_no_sequences(eng):
    k = eng.upload(np.zeros((32, 64), np.float32))
    table, lens = eng.empty(0, 3, miburn.I32), eng.empty(0, 1, miburn.I32)
    out = eng.paged_attention(eng.empty(0, 128), k, k, table, lens, 2, 2, 16, 0.125)
    assert eng.metadata(out) == (0, 128, F32)
    eng.sync()


def test_attention_shared_pages_and_repeated_rows(eng):
    """Sequences that share a prefix's pages, and the positions of one
    sequence's new rows as rows of one table."""
    rng = np.random.default_rng(12)
    c = Cache(rng, [64, 70, 0, 0, 0], 2, 64, 16, BF16, width=8)
    c.table[1, :4] = c.table[0, :4]      # one prefix
    c.table[2:] = c.table[1]
    c.lens[2:] = [67, 68, 69]            # the rows before sequence 1's last
    attend_check(eng, c.up(eng), 8)


@pytest.mark.parametrize("ce", [F32, BF16])
@pytest.mark.parametrize("prompts,heads,kv,d,page", [([300], 4, 2, 32, 16), ([700, 5, 460], 3, 1, 64, 48),
                                                     ([1300], 2, 1, 16, 16)])
def test_attention_of_whole_prompts(eng, prompts, heads, kv, d, page, ce):
    """A prompt's positions as rows: its table row repeated, each position
    with its own length."""
    rng = np.random.default_rng(sum(prompts))
    one = Cache(rng, prompts, kv, d, page, ce).poison()
    table, lens = [], []
    for s, n in enumerate(prompts):
        table += [one.table[s]] * n
        lens += range(1, n + 1)
    one.table, one.lens = np.array(table, np.int32), lens
    attend_check(eng, one.up(eng), heads)


def test_attention_equals_contiguous_cache(eng):
    """One slot a sequence: mi_attention_rows_at's values within both
    kernels' tolerances."""
    rng = np.random.default_rng(13)
    batch, heads, kv, d, maxc, n = 4, 9, 3, 64, 640, 577
    k, v = (rng.standard_normal((batch * kv * maxc, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((batch, heads * d)).astype(np.float32)
    kid, vid, qid = eng.upload(k), eng.upload(v), eng.upload(q)
    table = eng.upload_i32(np.arange(batch).reshape(-1, 1))
    lens = eng.upload_i32(np.full((batch, 1), n))
    a = eng.download(eng.attention_rows(qid, kid, vid, batch, 1, heads, kv, n - 1, 0.125))
    b = eng.download(eng.paged_attention(qid, kid, vid, table, lens, heads, kv, maxc, 0.125))
    c = Cache(rng, [n] * batch, kv, d, maxc, F32, spare=0)
    c.table[:, 0], c.k, c.v = np.arange(batch), k, v
    _, tol = attend64(c, q, heads, 0.125)
    assert np.all(np.abs(a.astype(np.float64) - b) <= 2 * tol)


@pytest.mark.parametrize("ce", [F32, BF16])
def test_attention_large_scores(eng, ce):
    """Scores in the hundreds: nearly all weight on one position."""
    rng = np.random.default_rng(14)
    attend_check(eng, Cache(rng, [300, 5], 2, 64, 16, ce).poison().up(eng), 4, scale=30.0)


@pytest.mark.parametrize("ce", [F32, BF16])
def test_attention_nan_and_lowest_scores(eng, ce):
    """A NaN key spoils the rows of its kv head of its sequence, a NaN value
    its column of them, and nothing else; a position whose score is far below
    the others' has no weight."""
    rng = np.random.default_rng(15)
    c = Cache(rng, [100, 100, 100], 2, 64, 16, ce).poison()
    c.k[c.row(1, 50, 0), 3] = np.nan
    c.v[c.row(1, 60, 1), 7] = np.nan
    low = c.row(2, 40, 0)
    c.k[low] = 0
    c.k[low, 5] = -1e30
    c.up(eng)
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    q[2, :, 5] = 1.0
    got = eng.download(eng.paged_attention(eng.upload(q.reshape(3, -1)), c.kid, c.vid, c.tid, c.lid, 4, 2, 16, 0.125))
    got = got.reshape(3, 4, 64)
    nan = np.isnan(got)
    assert nan[1, :2].all() and nan[1, 2:, 7].all()
    nan[1, :2], nan[1, 2:, 7] = False, False
    assert not nan.any()
    rows = c.rows(2, 0)
    rows = rows[rows != low]
    k, v = c.k[rows].astype(np.float64), c.v[rows].astype(np.float64)
    for h in (0, 1):
        qh = q[2, h].astype(np.float64)
        x = k @ qh * 0.125
        p = np.exp(x - x.max())
        p /= p.sum()
        tol = U * (4 * 72 * (np.abs(k) @ np.abs(qh) * 0.125).max() + 264) * (p @ np.abs(v))
        assert np.all(np.abs(got[2, h] - p @ v) <= tol)


@pytest.mark.parametrize("ce", [F32, BF16])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_attention_of_large_pools(eng, d, ce):
    """Pools larger than the last cache, NaN outside the sequences' pages;
    rows that begin with their neighbour's page and rows that do not."""
    rng = np.random.default_rng(d)
    kv, page, lens = 2, 16, [700, 0, 33, 1, 130, 130]
    small = Cache(rng, lens, kv, d, page, ce)
    small.table[5] = small.table[4]
    rows = kv * page
    pages = (80 << 20) // (rows * d * (4 if ce == F32 else 2))
    pools = []
    place = rng.permutation(pages)[:small.pages]
    for host in (small.k, small.v):
        src = put(eng, host, ce)[0]
        pool = eng.fill(pages * rows, d, ce, 0x7FC00000 if ce == F32 else 0x7FC0)
        for at in range(small.pages):
            eng.copy_into4(pool, int(place[at]) * rows * d, (0, 0, d, 1), src, at * rows * d, (0, 0, d, 1), (1, 1, rows, d))
        pools.append(pool)
    table = np.where((small.table >= 0) & (small.table < small.pages), place[np.clip(small.table, 0, small.pages - 1)], -1)
    heads, scale = 6, float(np.float32(d ** -0.5))
    q = rng.standard_normal((len(lens), heads * d)).astype(np.float32)
    tid, lid = eng.upload_i32(table), eng.upload_i32(np.array(lens).reshape(-1, 1))
    got = eng.download(eng.paged_attention(eng.upload(q), pools[0], pools[1], tid, lid, heads, kv, page, scale))
    want, tol = attend64(small, q, heads, scale)
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol)
    for p in pools:
        eng.free(p)
    eng.sync()


def test_attention_past_32_bits(eng):
    """Element offsets of a pool past 2^31 (keys and values one buffer)."""
    kv, d, page, n = 8, 128, 64, 100
    rows = kv * page
    pages = (1 << 31) // (rows * d) + 40
    pool = eng.fill(pages * rows, d, BF16, 0x7FC0)  # NaN throughout
    rng = np.random.default_rng(16)
    c = Cache(rng, [n], kv, d, page, BF16, spare=0)
    small = put(eng, c.k, BF16)[0]
    far = [pages - 2, pages - 39]
    for i, p in enumerate(far):
        eng.copy_into4(pool, p * rows * d, (0, 0, d, 1), small, int(c.table[0, i]) * rows * d, (0, 0, d, 1), (1, 1, rows, d))
    q = rng.standard_normal((1, 8 * d)).astype(np.float32)
    scale = float(np.float32(d ** -0.5))
    table, lens = eng.upload_i32(np.array([far])), eng.upload_i32(np.array([[n]]))
    got = eng.download(eng.paged_attention(eng.upload(q), pool, pool, table, lens, 8, kv, page, scale))
    c.v = c.k
    want, tol = attend64(c, q, 8, scale)
    assert np.all(np.abs(got.astype(np.float64) - want) <= tol)
    # One more position appended there.
    other = eng.fill(pages * rows, d, BF16, 0)
    x = rng.standard_normal((1, 24 * d)).astype(np.float32)
    cos, sin = rope_tables(n + 1, d)
    eng.qkv_rope_paged(eng.upload(x), eng.upload(cos), eng.upload(sin), table, eng.upload_i32(np.array([[n + 1]])), 0, 8,
                       kv, page, pool, other)
    back = eng.copy_strided(other, kv, d, (far[1] * rows + n % page) * d, page * d, 1)
    want_v = x.reshape(24, d)[16:]
    assert np.array_equal(eng.download(back), miburn.bf16_bits(want_v).reshape(8, d))
    assert eng.download(eng.reduce_all(eng.cast_float(back, F32), miburn.R_MAX))[0, 0] != 0
    eng.free(pool)
    eng.free(other)
    eng.sync()


@pytest.mark.parametrize("spoil", ["page", "page_high", "long", "negative"])
def test_attention_out_of_range(eng, spoil):
    """Reported at the next wait; the other sequences' rows are right."""
    rng = np.random.default_rng(17)
    c = Cache(rng, [40, 50, 60], 2, 64, 16, BF16, width=4)
    good = [40, 50, 60]
    if spoil == "page":
        c.table[1, 1] = -1
    elif spoil == "page_high":
        c.table[1, 1] = c.pages
    else:
        c.lens[1] = 65 if spoil == "long" else -1
    c.up(eng)
    q = rng.standard_normal((3, 4 * 64)).astype(np.float32)
    out = eng.paged_attention(eng.upload(q), c.kid, c.vid, c.tid, c.lid, 4, 2, 16, 0.125)
    with pytest.raises(miburn.MiError) as e:
        eng.sync()
    assert e.value.kind == "DOMAIN"
    got = eng.download(out)
    c.lens = [good[0], 0, good[2]]
    want, tol = attend64(c, q, 4, 0.125)
    for s in (0, 2):
        assert np.all(np.abs(got[s].astype(np.float64) - want[s]) <= tol[s])
    if spoil in ("long", "negative"):
        assert not got[1].any()


# ------------------------------------------------------------------ refusals


def test_refusals(eng):
    kv, d, page, heads = 2, 64, 16, 4
    k = eng.upload(np.zeros((4 * kv * page, d), np.float32))
    v = eng.upload(np.zeros((4 * kv * page, d), np.float32))
    k16 = eng.upload_bf16(np.zeros((4 * kv * page, d), np.uint16))
    odd = eng.upload(np.zeros((4 * kv * page, 48), np.float32))
    ints = eng.upload_i32(np.zeros((4 * kv * page, d)))
    table, lens = eng.upload_i32(np.zeros((2, 3))), eng.upload_i32(np.ones((2, 1)))
    ftable, flens = eng.upload(np.zeros((2, 3))), eng.upload(np.ones((2, 1)))
    lens3, starts = eng.upload_i32(np.ones((3, 1))), eng.upload_i32(np.arange(3).reshape(-1, 1))
    wide = eng.empty(2, 1 << 27, miburn.I32)
    q = eng.upload(np.zeros((2, heads * d)))
    qkv = eng.upload(np.zeros((2, (heads + 2 * kv) * d)))
    qkv5 = eng.upload(np.zeros((5, (heads + 2 * kv) * d)))
    cos, sin = (eng.upload(t) for t in rope_tables(48, d))
    short = eng.upload(np.zeros((47, d)))
    before = eng.report()["live_buffers"]

    def refused(kind, fn, *a):
        with pytest.raises(miburn.MiError) as e:
            fn(*a)
        assert e.value.kind == kind, e.value

    att, app = eng.paged_attention, eng.qkv_rope_paged
    for kind, a in [
        ("ARG", (q, k, k16, table, lens, heads, kv, page, 1.0)),
        ("ARG", (q, ints, ints, table, lens, heads, kv, page, 1.0)),
        ("UNSUPPORTED", (q, odd, odd, table, lens, heads, kv, page, 1.0)),
        ("ARG", (q, k, odd, table, lens, heads, kv, page, 1.0)),
        ("ARG", (q, k, v, ftable, lens, heads, kv, page, 1.0)),
        ("ARG", (q, k, v, table, flens, heads, kv, page, 1.0)),
        ("ARG", (q, k, v, table, lens3, heads, kv, page, 1.0)),
        ("ARG", (q, k, v, table, lens, 5, kv, page, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, 0, page, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, 3, page, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, kv, 0, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, kv, 2**40, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, kv, 24, 1.0)),   # not whole pages
        ("ARG", (q, k, v, table, lens, 8, kv, page, 1.0)),     # q of other heads
        ("ARG", (ints, k, v, table, lens, heads, kv, page, 1.0)),
        ("ARG", (q, k, v, table, lens, heads, kv, page, 1.0, miburn.I32)),
        ("UNSUPPORTED", (q, k, v, wide, lens, heads, kv, page, 1.0)),
        ("ID", (q, k, v, 10**9, lens, heads, kv, page, 1.0)),
    ]:
        refused(kind, att, *a)
    for kind, a in [
        ("ARG", (qkv, cos, sin, table, lens, 0, heads, kv, page, k, k16)),
        ("ARG", (qkv, cos, sin, table, lens, 0, heads, kv, page, k, k)),
        ("UNSUPPORTED", (qkv, cos, sin, table, lens, 0, heads, kv, page, odd, odd)),
        ("ARG", (qkv, cos, short, table, lens, 0, heads, kv, page, k, v)),
        ("ARG", (qkv, odd, odd, table, lens, 0, heads, kv, page, k, v)),
        ("ARG", (qkv5, cos, sin, table, lens, 0, heads, kv, page, k, v)),  # rows without starts
        ("ARG", (qkv, cos, sin, table, lens, lens, heads, kv, page, k, v)),  # starts of 2
        ("ARG", (qkv, cos, sin, table, lens, cos, heads, kv, page, k, v)),
        ("ARG", (qkv, cos, sin, table, lens, 0, 6, kv, page, k, v)),
        ("ARG", (ints, cos, sin, table, lens, 0, heads, kv, page, k, v)),
        ("ARG", (qkv, cos, sin, table, lens, 0, heads, kv, page, k, v, miburn.BOOL)),
        ("ID", (qkv, cos, sin, table, lens, 10**9, heads, kv, page, k, v)),
    ]:
        refused(kind, app, *a)
    assert eng.report()["live_buffers"] == before, "a refused call left a buffer"
    eng.free(app(qkv, cos, sin, table, lens, starts, heads, kv, page, k, v))
    eng.sync()


# ------------------------------------------------------------- other calls


def test_trace_replays_at_any_lengths(eng):
    """A decode step's append and attention captured once, replayed as the
    sequences grow and one falls idle: each replay the eager call's bits."""
    rng = np.random.default_rng(18)
    heads, kv, d, page, S = 9, 3, 64, 16, 3
    start = [15, 700, 31]
    c = Cache(rng, [40, 740, 60], kv, d, page, BF16).up(eng)
    pools = [eng.upload_bf16(eng.download(i)) for i in (c.kid, c.vid)]  # the eager run's
    cos, sin = (eng.upload(t) for t in rope_tables(800, d))
    x = eng.upload(np.zeros((S, (heads + 2 * kv) * d)))
    lens = eng.upload_i32(np.array(start).reshape(-1, 1))
    scale = float(np.float32(d ** -0.5))

    def step(kp, vp):
        q = eng.qkv_rope_paged(x, cos, sin, c.tid, lens, 0, heads, kv, page, kp, vp)
        o = eng.paged_attention(q, kp, vp, c.tid, lens, heads, kv, page, scale)
        eng.free(q)
        return o
    eng.begin_trace()
    out = step(c.kid, c.vid)
    trace = eng.end_trace()
    for i in range(6):
        xs = rng.standard_normal((S, (heads + 2 * kv) * d)).astype(np.float32)
        ls = np.array([[n + i] for n in start], np.int32)
        if i == 3:
            ls[1] = 0
        got, = eng.run_trace(trace, {x: xs, lens: ls}, [out])
        o = step(*pools)
        assert np.array_equal(bits(got), bits(eng.download(o))), i
        eng.free(o)
        eng.sync()
    for a, b in zip((c.kid, c.vid), pools):
        assert np.array_equal(eng.download(a), eng.download(b))
    eng.release_trace(trace)


@pytest.mark.parametrize("seqs,most", [(100, 700), (300, 700), (300, 300)])
def test_trace_of_many_sequences_replays_at_any_lengths(eng, seqs, most):
    """The attention of many sequences captured once: lengths that change
    between replays, eager calls of another size in between."""
    rng = np.random.default_rng(seqs + most)
    c = Cache(rng, [most] * seqs, 1, 32, 16, BF16).up(eng)
    few = Cache(rng, [3000, 40], 1, 32, 16, F32).poison().up(eng)
    q, fq = (eng.upload(rng.standard_normal((n, 64))) for n in (seqs, 2))
    lens = eng.upload_i32(np.zeros((seqs, 1)))
    eng.begin_trace()
    out = eng.paged_attention(q, c.kid, c.vid, c.tid, lens, 2, 1, 16, 0.25)
    trace = eng.end_trace()
    other = eng.download(eng.paged_attention(fq, few.kid, few.vid, few.tid, few.lid, 2, 1, 16, 0.25))
    for turn in range(5):
        ls = rng.integers(0, most + 1, (seqs, 1)).astype(np.int32)
        if turn == 2:
            ls[:] = 0
        if turn == 3:
            ls[:] = 1
            ls[seqs // 2] = most
        got, = eng.run_trace(trace, {lens: ls}, [out])
        o = eng.paged_attention(fq, few.kid, few.vid, few.tid, few.lid, 2, 1, 16, 0.25)
        assert np.array_equal(bits(eng.download(o)), bits(other))
        c.lens = ls[:, 0].tolist()
        want, tol = attend64(c, eng.download(q), 2, 0.25)
        assert np.all(np.abs(got - want) <= tol), turn
        eager = eng.paged_attention(q, c.kid, c.vid, c.tid, lens, 2, 1, 16, 0.25)
        assert np.array_equal(bits(got), bits(eng.download(eager))), turn
        eng.free(o)
        eng.free(eager)
        eng.sync()
    eng.release_trace(trace)


def test_two_traces_and_eager_calls_share_the_scratch(eng):
    """Two captured calls of unequal sizes and eager ones between them."""
    rng = np.random.default_rng(19)
    small = Cache(rng, [300, 7], 2, 64, 16, F32).poison().up(eng)
    large = Cache(rng, [9000] * 4, 2, 64, 16, F32).poison().up(eng)
    q = [eng.upload(rng.standard_normal((len(c.lens), 8 * 64))) for c in (small, large)]

    def call(i, c):
        return eng.paged_attention(q[i], c.kid, c.vid, c.tid, c.lid, 8, 2, 16, 0.125)
    want = [eng.download(call(i, c)) for i, c in enumerate((small, large))]
    traces, outs = [], []
    for i, c in enumerate((small, large)):
        eng.begin_trace()
        outs.append(call(i, c))
        traces.append(eng.end_trace())
    for turn in range(3):
        for i in ((0, 1), (1, 0), (0, 1))[turn]:
            got, = eng.run_trace(traces[i], {}, [outs[i]])
            assert np.array_equal(bits(got), bits(want[i]))
            assert np.array_equal(bits(eng.download(call(1 - i, (small, large)[1 - i]))), bits(want[1 - i]))
    for t in traces:
        eng.release_trace(t)


def test_repeats_are_bit_identical_and_calls_from_threads(eng):
    rng = np.random.default_rng(20)
    c = Cache(rng, [2000, 1, 0, 513, 77], 2, 128, 16, BF16).poison().up(eng)
    qid = eng.upload(rng.standard_normal((5, 8 * 128)))

    def call():
        return eng.download(eng.paged_attention(qid, c.kid, c.vid, c.tid, c.lid, 8, 2, 16, 0.1))
    want, got = call(), []
    threads = [threading.Thread(target=lambda: got.append(call())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(np.array_equal(bits(g), bits(want)) for g in got)


# ------------------------------------------------------------- a whole model


@pytest.mark.parametrize("cache", [F32, BF16])
def test_serving_run_against_the_decoder(eng, cache):
    """Prompts of unequal lengths and greedy decode steps of a small decoder
    on the paged operators -- append, attention, log probabilities -- against
    the harness's forward, a sequence at a time.  Prompts go in one call, a
    table row a position.  Every step's logits are within 2e-2 (the model
    bound of the decoder's own tests); with a BF16 cache the harness runs its
    performance contract's, which rounds as much again."""
    cfg = dict(vocab=512, hidden=128, layers=3, heads=4, kv_heads=2, head_dim=32, intermediate=256,
               rope_theta=1e4, eps=1e-5)
    heads, kv, d, L = 4, 2, 32, 3
    rng = np.random.default_rng(21)
    prompts = [rng.integers(0, 512, n).astype(np.int32) for n in (5, 33, 16)]
    steps, page = 4, 16
    total = [len(p) + steps for p in prompts]
    m = miburn.Llama(eng, cfg, max_ctx=64, max_batch=1, seed=7, init_std=0.08)
    par = {n: [m.param(n, i) for i in range(L)] for n in ("attn_norm", "wq", "wk", "wv", "wo", "mlp_norm", "wgate", "wup",
                                                      "wdown")}
    embed, final = m.param("embed"), m.param("final_norm")
    wqkv = [eng.upload_bf16(np.concatenate([eng.download(par[n][i]) for n in ("wq", "wk", "wv")])) for i in range(L)]
    caches = [Cache(np.random.default_rng(22), total, kv, d, page, cache) for _ in range(L)]
    for c in caches:
        c.k[:], c.v[:] = np.nan, np.nan
        c.up(eng)
    cos, sin = (eng.upload(t) for t in rope_tables(64, d, 1e4))
    table = caches[0].table

    def forward(ids, lens, news):
        """Logits of every new row: ids and each sequence's new rows."""
        rows = sum(news)
        lid = eng.upload_i32(np.array(lens).reshape(-1, 1))
        starts = eng.upload_i32(np.concatenate([[0], np.cumsum(news)]).reshape(-1, 1))
        seq = np.repeat(np.arange(len(news)), news)
        rlen = np.concatenate([np.arange(n - w, n) + 1 for n, w in zip(lens, news)])
        rt, rl = eng.upload_i32(table[seq]), eng.upload_i32(rlen.reshape(-1, 1))
        x = eng.select_rows_as(embed, eng.upload_i32(np.array(ids).reshape(-1, 1)), F32)
        for i, c in enumerate(caches):
            qkv = eng.matmul_dram(eng.rms_norm(x, par["attn_norm"][i], 1e-5), False, wqkv[i], True)
            q = eng.qkv_rope_paged(qkv, cos, sin, eng.upload_i32(c.table), lid, starts, heads, kv, page, c.kid, c.vid)
            o = eng.paged_attention(q, c.kid, c.vid, rt, rl, heads, kv, page, float(np.float32(d ** -0.5)))
            x = eng.linear(o, par["wo"][i], True, 0, x)
            n = eng.rms_norm(x, par["mlp_norm"][i], 1e-5)
            h = eng.eltwise_op_as("SILU_MUL", eng.matmul_dram(n, False, par["wgate"][i], True),
                                  eng.matmul_dram(n, False, par["wup"][i], True))
            x = eng.linear(h, par["wdown"][i], True, 0, x)
        assert eng.metadata(x)[0] == rows
        return eng.matmul_dram(eng.rms_norm(x, final, 1e-5), False, embed, True)

    def near(got, want, what):
        assert np.abs(got - want).max() <= 2e-2 * np.abs(want).max(), what

    lens, news = [len(p) for p in prompts], [len(p) for p in prompts]
    ids = np.concatenate(prompts)
    texts = [list(p) for p in prompts]
    for step in range(steps):
        logits = forward(ids, lens, news)
        last = np.cumsum(news) - 1
        rows = eng.select_rows(logits, eng.upload_i32(last.reshape(-1, 1)))
        z = eng.download(rows)
        pick = eng.download(eng.argmax_row(rows)).ravel()
        r = eng.token_logprobs(rows, eng.upload_i32(pick.reshape(-1, 1)), 1.0, 3)
        assert np.array_equal(eng.download(r.top_ids)[:, 0], pick)
        assert np.array_equal(eng.download(r.logp), eng.download(r.top_logp)[:, :1])
        z64 = z.astype(np.float64)
        lse = np.log(np.exp(z64 - z64.max(1, keepdims=True)).sum(1)) + z64.max(1)
        assert np.allclose(eng.download(r.logp).ravel(), z64[np.arange(3), pick] - lse, rtol=0, atol=2e-5)
        for s, t in enumerate(texts):
            m.reset()
            near(z[s], eng.download(m.forward(np.array([t], np.int32)))[0], (step, s))
            t.append(int(pick[s]))
        ids, lens, news = pick, [n + 1 for n in lens], [1, 1, 1]
    m.close()
    eng.sync()
