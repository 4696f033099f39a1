"""mi_token_logprobs and its backward on the device, against float64.

Tolerances, with u = 2^-24, z = scale x, m = max z, d = z - m, e = e^d,
S = sum e, p = e / S, K = cols / 256 + 64 (no sum chains more additions): z and
m are each one rounding of a product (u |z|, u |m|) and d one more, so an e is
off by u (|z| + |m| + |d| + 4) of itself, and S by the p-weighted mean of that
and K u: eS.  lse = m + ln S is off by u (2 |m| + |lse| + 4) + eS, and logp =
z_t - lse by that and u (2 |z_t| + |logp|).  entropy = ln S - T / S is off by
eS + 2 u ln S and by sum p |d| (u (|z| + |m| + 2 |d| + 2 K + 16)) +
u sum p (|z| + |m| + |d|) + eS sum p |d|.
"""
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


def put(eng, x, elem):
    x = np.ascontiguousarray(x, np.float32)
    if elem == F32:
        return eng.upload(x), x
    b = miburn.bf16_bits(x)
    return eng.upload_bf16(b.reshape(x.shape)), miburn.bf16_to_f32(b).reshape(x.shape)


def column(eng, v):
    return eng.upload_i32(np.asarray(v, np.int32).reshape(-1, 1))


def order(x):
    """Columns of each row: the largest value first, a NaN above all, the
    lowest column among equals."""
    key = np.where(np.isnan(x), np.inf, x.astype(np.float64))
    top = np.isnan(x).astype(np.int64)
    cols = np.broadcast_to(np.arange(x.shape[1]), x.shape)
    return np.lexsort((cols, -key, -top), axis=1)


def stats64(x, scale):
    """(z, p, lse, entropy, tolerance of lse, of entropy), finite rows."""
    z = x.astype(np.float64) * float(np.float32(scale))
    m = z.max(1, keepdims=True)
    d = z - m
    e = np.exp(d)
    S = e.sum(1, keepdims=True)
    p = e / S
    with np.errstate(invalid="ignore"):
        ad, az = np.where(p > 0, np.abs(d), 0), np.where(p > 0, np.abs(z), 0)
    lnS = np.log(S[:, 0])
    K = x.shape[1] / 256 + 64
    off = az + np.abs(m) + ad
    eS = U * ((p * (off + 4)).sum(1) + K)
    lse, mean = m[:, 0] + lnS, (p * ad).sum(1)
    tl = U * (2 * np.abs(m[:, 0]) + np.abs(lse) + 4) + eS
    te = eS + 2 * U * lnS + U * (p * ad * (off + ad + 2 * K + 16)).sum(1) + U * (p * off).sum(1) + eS * mean
    return z, p, lse, lnS + mean, tl, te


def check(eng, x, elem, scale, top, targets=None, with_targets=True):
    xid, x = put(eng, x, elem)
    rows = x.shape[0]
    t = np.random.default_rng(rows).integers(0, x.shape[1], rows) if targets is None else np.asarray(targets)
    r = eng.token_logprobs(xid, column(eng, t) if with_targets else 0, scale, top)
    z, p, lse, ent, tl, te = stats64(x, scale)
    got = eng.download(r.lse)[:, 0]
    assert np.all(np.abs(got - lse) <= tl), np.abs(got - lse).max()
    got = eng.download(r.entropy)[:, 0]
    assert np.all(np.abs(got - ent) <= te), (np.abs(got - ent) / te).max()
    at = np.arange(rows)
    if with_targets:
        got = eng.download(r.logp)[:, 0].astype(np.float64)
        want = z[at, t] - lse
        with np.errstate(invalid="ignore"):
            tol = tl + U * (2 * np.abs(z[at, t]) + np.abs(want))
            assert np.all((np.abs(got - want) <= tol) | (got == want))
    else:
        assert r.logp == 0
    if top:
        ids = eng.download(r.top_ids)
        best = order(x)[:, :top]
        assert ids.dtype == np.int32 and np.array_equal(ids, best)
        got = eng.download(r.top_logp).astype(np.float64)
        zt = np.take_along_axis(z, best, 1)
        want = zt - lse[:, None]
        with np.errstate(invalid="ignore"):
            tol = tl[:, None] + U * (2 * np.abs(zt) + np.abs(want))
            assert np.all((np.abs(got - want) <= tol) | (got == want))
    else:
        assert r.top_logp == 0 and r.top_ids == 0
    for i in r:
        if i:
            eng.free(i)
    eng.sync()


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("rows,cols,top", [
    (1, 1, 1), (3, 2, 2), (5, 31, 31), (4, 64, 32), (7, 255, 5), (2, 256, 32), (9, 257, 20), (300, 1000, 5),
    (2, 8192, 32), (3, 8193, 1), (1, 49152, 20), (33, 16385, 8), (2, 40001, 32), (1, 160001, 5), (600, 4099, 3),
    (1, 500000, 32), (300, 100001, 7), (20, 70000, 32), (130, 99999, 3), (3, 49152, 32), (1, 12289 * 4, 9),
])
def test_shapes(eng, rows, cols, top, elem):
    rng = np.random.default_rng(rows + cols)
    check(eng, rng.standard_normal((rows, cols)) * 3, elem, 1.0, top)


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("scale", [1 / 0.7, 0.5, 8.0, 1e-3])
def test_scales_and_no_targets(eng, scale, elem):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 5003)) * 4
    check(eng, x, elem, scale, 0)
    check(eng, x, elem, scale, 20, with_targets=False)


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("cols", [40, 1000, 9001, 50001, 120001])
def test_ties(eng, cols, elem):
    """Equal logits: the lowest columns, wherever they lie."""
    rng = np.random.default_rng(cols)
    few = rng.integers(-3, 4, (6, cols)).astype(np.float32)
    few[0] = 2.5                         # all alike
    few[1] = np.where(np.arange(cols) < cols - 7, -1.0, 1.0)  # the best ones last
    few[2] = np.where(rng.random(cols) < 0.5, 0.0, -0.0)      # 0 and -0 are equal
    few[3] = -np.arange(cols)            # descending
    few[4] = np.arange(cols)             # ascending
    check(eng, few, elem, 1.0, 32)


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("cols", [4001, 9000, 33001, 49152, 98304])
def test_as_many_equal_columns_as_there_is_room_for(eng, cols, elem):
    """Around 1024 columns of the largest value, spread, at the front and at
    the end, and a few above them."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((15, cols)) - 8
    for r, n in enumerate((1022, 1023, 1024, 1025, 1056)):
        x[r, rng.permutation(cols)[:n]] = 2
        x[5 + r, :n] = 2
        x[10 + r, cols - n:] = 2
        x[10 + r, rng.permutation(cols)[:3]] = 3
    check(eng, x, elem, 1.0, 32)


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("cols", [100, 3001, 50000, 120000])
def test_masked_logits(eng, cols, elem):
    """-inf in all places but some, and values near the type's lowest."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((5, cols)).astype(np.float32)
    x[0, 1:] = -np.inf
    x[1, :-1] = -np.inf
    x[2, rng.random(cols) < 0.95] = -np.inf
    x[3, rng.random(cols) < 0.5] = -3.3e38
    x[3, 17] = 1.0
    x[4] = -3.3e38                      # all at the lowest values: uniform
    check(eng, x, elem, 1.0, 32, targets=[0, 0, 17, 17, 3])


@pytest.mark.parametrize("elem,lanes", [(BF16, 8), (F32, 4)])
def test_masked_to_a_few_threads_columns(eng, elem, lanes):
    """What a mask leaves lies in the columns of a few threads, more of them
    than a block holds as candidates (columns in chunks of `lanes`, a chunk a
    thread of 512)."""
    rng = np.random.default_rng(lanes)
    rows, cols = 512, 2000 * lanes
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    x[:, (np.arange(cols) // lanes) % 512 >= 40 * 8 // lanes] = -np.inf
    x[3:] = x[:1]
    check(eng, x, elem, 1.0, 32, targets=np.zeros(rows, np.int64))


@pytest.mark.parametrize("elem", [F32, BF16])
@pytest.mark.parametrize("cols", [77, 20000, 100003])
def test_empty_and_not_finite_rows(eng, cols, elem):
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((5, cols)).astype(np.float32)
    x[0] = -np.inf                      # nothing left
    x[1, cols // 2] = np.nan
    x[2, 5] = np.inf
    x[3, 9], x[3, 3] = np.nan, np.nan
    xid, x = put(eng, x, elem)
    r = eng.token_logprobs(xid, column(eng, [1, 2, 3, 4, 5]), 1.0, 4)
    logp, lse, ent, tl, ids = (eng.download(i) for i in r)
    assert lse[0, 0] == -np.inf and logp[0, 0] == -np.inf and ent[0, 0] == 0
    assert np.all(tl[0] == -np.inf) and np.array_equal(ids[0], [0, 1, 2, 3])
    for row in (1, 2, 3):
        assert np.isnan(lse[row, 0]) and np.isnan(ent[row, 0]) and np.isnan(logp[row, 0])
    assert np.isfinite(logp[4, 0])
    assert np.array_equal(ids, order(x)[:, :4])
    eng.sync()


def test_far_logits(eng):
    """A large common offset, and one logit far above the others."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 5000)).astype(np.float32)
    check(eng, x + 3e4, F32, 1.0, 5)
    check(eng, x - 3e4, F32, 1.0, 5)
    x[:, 77] = 500
    check(eng, x, F32, 1.0, 5, targets=[77, 0, 77])


@pytest.mark.parametrize("targets", [[0, -1, 2], [0, 50, 2], [0, -2**31, 2]])
def test_targets_out_of_range(eng, targets):
    x = np.random.default_rng(7).standard_normal((3, 50)).astype(np.float32)
    xid, tid = eng.upload(x), column(eng, targets)
    r = eng.token_logprobs(xid, tid)
    with pytest.raises(miburn.MiError) as e:
        eng.sync()
    assert e.value.kind == "DOMAIN"
    logp = eng.download(r.logp)[:, 0]
    _, _, lse, _, tl, _ = stats64(x, 1.0)
    assert logp[1] == 0 and np.all(np.abs(logp[[0, 2]] - (x[[0, 2], [0, 2]] - lse[[0, 2]])) <= 2 * tl[[0, 2]])
    # Its logp passes no gradient; the entropy's stays.
    g, h = eng.upload(np.full((3, 1), 2.0)), eng.upload(np.full((3, 1), 0.5))
    a = eng.token_logprobs_backward(xid, tid, r.lse, r.entropy, g, h)
    with pytest.raises(miburn.MiError) as e:
        eng.sync()
    assert e.value.kind == "DOMAIN"
    b = eng.token_logprobs_backward(xid, 0, r.lse, r.entropy, 0, h)
    assert np.array_equal(eng.download(a)[1], eng.download(b)[1])


# ---------------------------------------------------------------- backward


def grad64(x, scale, t, lse, ent, g, h):
    """dlogits and its tolerance.  l = z - lse is off by u (|z| + |l|), p by
    that and 4 u of itself, the bracket's sums and products by 4 u of their
    terms: 6 covers them."""
    s = float(np.float32(scale))
    z = x.astype(np.float64) * s
    l = z - lse[:, None]
    p = np.exp(l)
    one = np.zeros_like(p)
    if t is not None:
        one[np.arange(len(t)), t] = 1
    with np.errstate(invalid="ignore"):
        pl = np.where(p > 0, p * (l + ent[:, None]), 0)
        pa = np.where(p > 0, p * (np.abs(l) + np.abs(ent)[:, None]), 0)
        el = np.where(p > 0, np.abs(z) + np.abs(l), 0)
    want = s * (g[:, None] * (one - p) - h[:, None] * pl)
    ag, ah = np.abs(g)[:, None], np.abs(h)[:, None]
    tol = s * U * ((ag * p + ah * pa) * (el + 12) + ah * p * el + 6 * ag * one) + 2.0**-140
    return want, tol


@pytest.mark.parametrize("elem,out", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 257), (40, 1000), (3, 8193), (1, 49152), (300, 509),
                                       (2, 40001)])
def test_backward(eng, rows, cols, elem, out):
    rng = np.random.default_rng(rows * 7 + cols)
    scale = 1.25
    xid, x = put(eng, rng.standard_normal((rows, cols)) * 3, elem)
    t = rng.integers(0, cols, rows)
    g, h = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    tid = column(eng, t)
    r = eng.token_logprobs(xid, tid, scale)
    gid, hid = eng.upload(g.reshape(-1, 1)), eng.upload(h.reshape(-1, 1))
    lse, ent = (eng.download(i)[:, 0].astype(np.float64) for i in (r.lse, r.entropy))
    for use_g, use_h in ((1, 1), (1, 0), (0, 1)):
        id_ = eng.token_logprobs_backward(xid, tid if use_g else 0, r.lse, r.entropy if use_h else 0,
                                          gid if use_g else 0, hid if use_h else 0, scale, out)
        assert eng.metadata(id_) == (rows, cols, out)
        got = eng.download(id_)
        got = miburn.bf16_to_f32(got).reshape(got.shape) if out == BF16 else got
        want, tol = grad64(x, scale, t if use_g else None, lse, ent, g * use_g, h * use_h)
        if out == BF16:
            tol = tol + 2.0**-8 * np.abs(want) + 2.0**-134
        off = np.abs(got.astype(np.float64) - want)
        assert np.all(off <= tol), (use_g, use_h, (off / tol).max())
        eng.free(id_)
    eng.sync()


def test_more_rows_than_one_launch_holds(eng):
    """A block a row is 2^24 - 1 blocks of 256 threads at most: the gradient
    takes the rows in two launches, the forward refuses them."""
    rows = 2**24 + 70
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, 2)).astype(np.float32)
    t = rng.integers(0, 2, rows).astype(np.int32)
    g = rng.standard_normal(rows).astype(np.float32)
    lse = np.logaddexp(x[:, 0], x[:, 1]).astype(np.float32)
    xid, tid = eng.upload(x), eng.upload_i32(t.reshape(-1, 1))
    lid, gid = eng.upload(lse.reshape(-1, 1)), eng.upload(g.reshape(-1, 1))
    out = eng.token_logprobs_backward(xid, tid, lid, 0, gid, 0)
    got = eng.download(out)
    for at in (slice(0, 1000), slice(2**23 - 500, 2**23 + 500), slice(rows - 1000, rows)):
        want, tol = grad64(x[at], 1.0, t[at], lse[at].astype(np.float64), np.zeros(len(t[at])), g[at], 0 * g[at])
        assert np.all(np.abs(got[at] - want) <= tol)
    before = eng.report()["live_buffers"]
    with pytest.raises(miburn.MiError) as e:
        eng.token_logprobs(xid, tid)
    assert e.value.kind == "UNSUPPORTED"
    assert eng.report()["live_buffers"] == before
    for i in (xid, tid, lid, gid, out):
        eng.free(i)
    eng.sync()


def test_backward_against_differences(eng):
    """sum(g logp + h entropy), its slope along random directions by central
    differences in 64 bits."""
    rng = np.random.default_rng(8)
    rows, cols, scale = 4, 300, 0.8
    x = (rng.standard_normal((rows, cols)) * 2).astype(np.float32)
    t = rng.integers(0, cols, rows)
    g, h = rng.standard_normal((2, rows)).astype(np.float32)
    xid, tid = eng.upload(x), column(eng, t)
    r = eng.token_logprobs(xid, tid, scale)
    d = eng.download(eng.token_logprobs_backward(xid, tid, r.lse, r.entropy, eng.upload(g.reshape(-1, 1)),
                                                 eng.upload(h.reshape(-1, 1)), scale)).astype(np.float64)

    def loss(x64):
        z = x64 * float(np.float32(scale))
        l = z - np.log(np.exp(z).sum(1, keepdims=True))
        return (g * l[np.arange(rows), t]).sum() - (h * (np.exp(l) * l).sum(1)).sum()
    for _ in range(5):
        v = rng.standard_normal((rows, cols))
        e = 1e-5
        slope = (loss(x + e * v) - loss(x - e * v)) / (2 * e)
        # The gradient's own tolerance (a few u per value) and the third
        # derivative's e^2.
        assert abs((d * v).sum() - slope) <= 1e-5 * np.abs(d * v).sum() + 1e-8


@pytest.mark.parametrize("elem", [F32, BF16])
def test_backward_masked_and_empty_rows(eng, elem):
    rng = np.random.default_rng(9)
    cols = 1001
    x = rng.standard_normal((4, cols)).astype(np.float32)
    x[0] = -np.inf
    x[1, ::2] = -np.inf
    x[2, 1:] = -np.inf
    x[3, 4] = np.nan
    xid, x = put(eng, x, elem)
    t = [5, 2, 0, 1]
    tid = column(eng, t)
    r = eng.token_logprobs(xid, tid)
    ones = eng.upload(np.ones((4, 1)))
    got = eng.download(eng.token_logprobs_backward(xid, tid, r.lse, r.entropy, ones, ones))
    want = np.zeros(cols, np.float32)
    want[5] = 1
    assert np.array_equal(got[0], want)
    lse, ent = (eng.download(i)[:3, 0].astype(np.float64) for i in (r.lse, r.entropy))
    w, tol = grad64(x[1:3], 1.0, t[1:3], lse[1:], ent[1:], np.ones(2), np.ones(2))
    assert np.all(np.abs(got[1:3] - w) <= tol)
    assert np.isnan(got[3]).any()
    eng.sync()


def test_equals_cross_entropy(eng):
    """On rows mi_log_softmax_ce takes: its picked values and gradient within
    both operators' tolerances."""
    rng = np.random.default_rng(10)
    x = (rng.standard_normal((50, 8192)) * 2).astype(np.float32)
    t = rng.integers(0, 8192, 50)
    xid, tid = eng.upload(x), column(eng, t)
    picked, d = eng.log_softmax_ce(xid, tid, 1 / 50)
    r = eng.token_logprobs(xid, tid)
    z, p, lse, ent, tl, _ = stats64(x, 1.0)
    assert np.all(np.abs(eng.download(picked) - eng.download(r.logp))[:, 0] <= 4 * tl + 4 * U * np.abs(z[np.arange(50), t]))
    g = eng.upload(np.full((50, 1), -1 / 50))
    mine = eng.download(eng.token_logprobs_backward(xid, tid, r.lse, 0, g, 0))
    _, tol = grad64(x, 1.0, t, lse, ent, np.full(50, 1 / 50), np.zeros(50))
    assert np.all(np.abs(mine - eng.download(d)) <= 4 * tol + p * 4 * tl[:, None] / 50)


# ------------------------------------------------------------- other calls


def test_refusals(eng):
    x, x1 = eng.upload(np.zeros((4, 40))), eng.upload(np.zeros((4, 1)))
    xi, none = eng.upload_i32(np.zeros((4, 40))), eng.empty(4, 0)
    t, t3 = column(eng, [0, 1, 2, 3]), column(eng, [0, 1, 2])
    r = eng.token_logprobs(x, t)
    before = eng.report()["live_buffers"]

    def refused(kind, fn, *a):
        with pytest.raises(miburn.MiError) as e:
            fn(*a)
        assert e.value.kind == kind, e.value
    f, b = eng.token_logprobs, eng.token_logprobs_backward
    for kind, a in [("ARG", (xi, t)), ("ARG", (none, t)), ("ARG", (x, t3)), ("ARG", (x, x1)), ("ARG", (x, t, 0.0)),
                    ("ARG", (x, t, -1.0)), ("ARG", (x, t, float("inf"))), ("ARG", (x, t, float("nan"))),
                    ("ARG", (x, t, 1.0, 33)), ("ARG", (x1, t, 1.0, 2)), ("ID", (10**9, t)), ("ID", (x, 10**9))]:
        refused(kind, f, *a)
    for kind, a in [("ARG", (x, t, r.lse, r.entropy, 0, 0)), ("ARG", (x, t, r.lse, 0, 0, 0)),
                    ("ARG", (x, 0, r.lse, 0, r.logp, 0)), ("ARG", (x, 0, r.lse, 0, 0, r.logp)),
                    ("ARG", (x, t3, r.lse, 0, r.logp, 0)), ("ARG", (x, t, t, 0, r.logp, 0)),
                    ("ARG", (x, t, r.lse, 0, x, 0)), ("ARG", (x, t, r.lse, 0, r.logp, 0, 0.0)),
                    ("ARG", (x, t, r.lse, 0, r.logp, 0, 1.0, miburn.I32)), ("ID", (x, t, 10**9, 0, r.logp, 0))]:
        refused(kind, b, *a)
    refused("ARG", lambda: eng._check(eng._lib.mi_token_logprobs(eng.ctx, x, 0, 1.0, 0, None, None, None, None, None)))
    assert eng.report()["live_buffers"] == before, "a refused call left a buffer"


def test_no_rows(eng):
    x, t = eng.empty(0, 40), eng.empty(0, 1, miburn.I32)
    r = eng.token_logprobs(x, t, 1.0, 3)
    assert eng.metadata(r.logp)[:2] == (0, 1) and eng.metadata(r.top_ids) == (0, 3, miburn.I32)
    d = eng.token_logprobs_backward(x, t, r.lse, r.entropy, r.logp, r.logp)
    assert eng.metadata(d)[:2] == (0, 40)
    eng.sync()


@pytest.mark.parametrize("rows,cols", [(1, 49152), (40, 5001), (2, 130001)])
def test_trace_replays(eng, rows, cols):
    """Forward and backward captured once, replayed on other logits, with an
    eager call of other sizes between: each replay the eager call's bits."""
    rng = np.random.default_rng(11)
    x, t = eng.upload(np.zeros((rows, cols))), column(eng, rng.integers(0, cols, rows))
    other = eng.upload(rng.standard_normal((3, 160001)))
    g = eng.upload(rng.standard_normal((rows, 1)))

    def step():
        r = eng.token_logprobs(x, t, 1.5, 20)
        return (*r, eng.token_logprobs_backward(x, t, r.lse, r.entropy, g, g, 1.5))
    eng.begin_trace()
    outs = step()
    trace = eng.end_trace()
    for i in range(4):
        got = eng.run_trace(trace, {x: rng.standard_normal((rows, cols)).astype(np.float32) * 3}, list(outs))
        for i_ in eng.token_logprobs(other, 0, 1.0, 5):
            if i_:
                eng.free(i_)
        eager = step()
        for a, b in zip(got, eager):
            assert np.array_equal(a.view(np.uint32), eng.download(b).view(np.uint32)), i
            eng.free(b)
        eng.sync()
    eng.release_trace(trace)
