"""Infinities and NaN that a row sees, in attention over the paged cache: a softmax weight is positive,
so an infinite value gives that infinity (NaN with one of the other sign), whatever its weight, its
place among the keys and the kernel that the batch's size selects."""
import math

import numpy as np
import pytest

import einsummable_amd as ea
from helpers import assert_bits_equal, stream_handle
from serving_oracle import NP, Paged, assert_within, attention64
from test_gpu_serving import OnDevice, dev

pytestmark = pytest.mark.gpu

F16, F32 = ea.F16, ea.F32


def attend(km, b, q, scale, shared=None):
    """[used tokens, heads, d]; the workspace holds NaN before the call."""
    import torch

    g = OnDevice(b)
    shared = b.shared if shared is None else shared
    need = km.prefix_attention_workspace(g.cache, b.n_seqs, b.tokens, shared)
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    d_q = dev(q.astype(NP[b.dtype]))
    d_o = torch.zeros_like(d_q)
    torch.cuda.synchronize()
    km.prefix_attention(g.cache, g.batch, shared, scale, stream_handle(), d_o.data_ptr(),
                        d_q.data_ptr(), (ws.data_ptr(), need) if need else None)
    torch.cuda.synchronize()
    return d_o.cpu().numpy()[:b.used].reshape(b.used, b.heads, b.d)


def queries(b, spread=1.0):
    return b.r.normal(0, spread, (b.tokens, b.heads, b.d)).astype(NP[b.dtype])


def put(b, cache, pos, element, value, seqs=None):
    """One element of every head's entry at a position (of all sequences that have it: a shared
    position may lie on a page of each)."""
    for s in range(b.n_seqs) if seqs is None else seqs:
        if pos < max(b.lens[s], b.shared):
            page, row = b.table[s, pos // b.page], pos % b.page
            if b.head_major:
                cache[page, :, row, element] = value
            else:
                cache[page, row, :, element] = value


def check(b, q, scale, got):
    with np.errstate(invalid="ignore"):
        want, bound = attention64(b, q, scale)
    want, bound = want[:b.used], bound[:b.used]
    for what, of in (("NaN", np.isnan), ("+inf", np.isposinf), ("-inf", np.isneginf)):
        differ = np.argwhere(of(got) != of(want))
        assert differ.size == 0, "%s: %d places, first %s" % (what, len(differ), differ[0])
    fine = np.isfinite(want)
    assert_within(got[fine], want[fine], bound[fine], "finite ones")


# heads, key heads, dim, page, new, lens, shared: rows of 16 and of 64 and 128 in the shared and in the
# own positions, prefixes that end inside a step of either kind
SHAPES = [
    (4, 2, 128, 8, [1] * 40, [200] * 40, 70),
    (4, 2, 64, 8, [1] * 15, [131] * 15, 70),
    (2, 2, 64, 8, [1, 2], [97, 140], 39),
    (8, 1, 128, 16, [5] * 8, [160] * 8, 70),
    (8, 1, 64, 16, [40, 33], [170, 121], 77),
    (4, 1, 200, 16, [30, 17], [90, 133], 33),
    (4, 4, 80, 24, [1] * 70, [90 + i for i in range(70)], 50)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "h%d-%d-d%d-t%d-s%d" %
                         (s[0], s[1], s[2], sum(s[4]), s[6]))
def test_visible_infinities_at_the_borders_of_parts(km, dtype, shape):
    shared = shape[-1]
    for n, pos in enumerate((shared - 1, shared, 0, shared // 32 * 32, min(shape[5]) - 1)):
        b = Paged(60 + n, dtype, *shape)
        q = queries(b)
        put(b, b.v, pos, 3, np.inf)
        put(b, b.v, pos, 4, -np.inf)
        put(b, b.v, pos, 5, np.nan)
        if pos > 9:                       # infinities of both signs
            put(b, b.v, pos, 6, np.inf)
            put(b, b.v, 9, 6, -np.inf)
        for part in (shared, 0):
            check(b, q, b.d ** -0.5, attend(km, b, q, b.d ** -0.5, part))


def test_visible_infinity_at_the_end_of_the_page_table(km):
    # 72 positions have a column, the sequences are longer
    for new in ([1, 2], [70, 3], [20, 20]):
        b = Paged(70, F16, 4, 1, 128, 24, new, [90, 85], extra_cols=0)
        b.table = np.ascontiguousarray(b.table[:, :3])
        q = queries(b)
        for s in range(2):
            b.v[b.table[s, 2], 23, :, 3] = np.inf
        check(b, q, 0.1, attend(km, b, q, 0.1))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new,lens,shared", [
    ([1], [400], 0), ([1], [400], 300), ([1] * 40, [400] * 40, 300), ([90], [400], 0),
    ([20] * 8, [333] * 8, 290)])
@pytest.mark.parametrize("gap", [30, 200])
def test_visible_infinity_of_small_weight(km, dtype, new, lens, shared, gap):
    """2^-30 of the largest weight, and one that underflows fp32: positive all the same."""
    b = Paged(71, dtype, 4, 1, 64, 16, new, lens, shared)
    q = np.zeros((b.tokens, 4, 64), NP[dtype])
    q[:, :, 0] = 1
    b.k[..., 0] = 0
    put(b, b.k, 40, 0, -gap)
    for v in (np.inf, -np.inf):
        put(b, b.v, 40, 3, v)
        check(b, q, math.log(2), attend(km, b, q, math.log(2)))
    # the whole prefix of small weight
    for pos in range(shared):
        put(b, b.k, pos, 0, -gap)
    if shared:
        check(b, q, math.log(2), attend(km, b, q, math.log(2)))


def test_rows_that_see_no_infinity_keep_every_bit(km):
    for shape in SHAPES:
        b = Paged(72, F16, *shape)
        q = queries(b)
        clean = attend(km, b, q, 0.1)
        s = b.n_seqs - 1
        put(b, b.v, b.lens[s] - 1, 3, np.inf, [s])
        got = attend(km, b, q, 0.1)
        last = b.used - 1
        assert_bits_equal(got[:last], clean[:last], "rows before the position")
        keep = [i for i in range(b.d) if i != 3]
        assert_bits_equal(got[last][:, keep], clean[last][:, keep], "other elements")
        assert np.isposinf(got[last, :, 3]).all()


# one own position each, behind the prefix: parts that hold a single key
ALONE = [(4, 2, 128, 8, [1] * 40, [71] * 40, 70), (4, 2, 64, 8, [1] * 3, [71] * 3, 70),
         (8, 1, 128, 16, [5] * 8, [75] * 8, 70)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shape", SHAPES + ALONE, ids=lambda s: "h%d-%d-d%d-t%d-s%d" %
                         (s[0], s[1], s[2], sum(s[4]), s[6]))
def test_nan_scores_reach_the_result(km, dtype, shape):
    """NaN in a query, and in keys that a row sees; all other rows keep every bit."""
    shared = shape[-1]
    for part in (shared, 0):
        b = Paged(73, dtype, *shape)
        q, scale = queries(b), b.d ** -0.5
        clean = attend(km, b, q, scale, part)
        bad = q.copy()
        bad[b.used // 2, 1, 5] = np.nan
        got = attend(km, b, bad, scale, part)
        assert np.isnan(got[b.used // 2, 1]).all()
        got[b.used // 2, 1] = clean[b.used // 2, 1]
        assert_bits_equal(got, clean, "NaN in a query")
        # the newest key of each sequence in turn; all keys of the first one's; a shared one
        for s in (0, b.n_seqs - 1):
            b = Paged(73, dtype, *shape)
            put(b, b.k, b.lens[s] - 1, 5, np.nan, [s])
            last = int(b.offsets[s + 1]) - 1
            got = attend(km, b, q, scale, part)
            assert np.isnan(got[last]).all()
            got[last] = clean[last]
            assert_bits_equal(got, clean, "NaN in the newest key")
        for pos in range(shared, b.lens[0]):
            put(b, b.k, pos, 0, np.nan, [0])
        got = attend(km, b, q, scale, part)
        b = Paged(73, dtype, *shape)
        put(b, b.k, shared - 1, 5, np.nan)
        assert np.isnan(got[b.new[0] - 1]).all()
        assert np.isnan(attend(km, b, q, scale, part)).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new,lens,shared", [
    ([1, 1, 2], [40, 1, 35], 0), ([1] * 40, [70] * 40, 33), ([70, 30], [70, 40], 0),
    ([9] * 8, [50] * 8, 33)])
def test_scores_of_minus_infinity(km, dtype, new, lens, shared):
    """Weight zero, as if there were no such key; a row that sees no other has no softmax: NaN."""
    b = Paged(74, dtype, 4, 1, 64, 1, new, lens, shared)
    q = queries(b)
    q[..., 0] = 1
    b.k[..., 0] = 0
    gone = Paged(74, dtype, 4, 1, 64, 1, new, lens, shared)
    gone.k[..., 0] = 0
    r = np.random.RandomState(0)
    for s in range(b.n_seqs):
        at = np.arange(shared, lens[s])
        at = at if s % 3 == 0 else r.permutation(at)[:at.size // 2]
        b.k[b.table[s, at], 0, :, 0] = -np.inf
        gone.table[s, at] = -1
    first = attend(km, b, q, 0.1)
    want, bound = attention64(gone, q, 0.1)
    for s in range(b.n_seqs):
        rows = slice(int(b.offsets[s]), int(b.offsets[s + 1]))
        sees = (gone.table[s, :lens[s]] >= 0).cumsum()[lens[s] - new[s]:lens[s]] > 0
        assert np.isnan(first[rows][~sees]).all()
        assert_within(first[rows][sees], want[rows][sees], bound[rows][sees], "keys of weight zero")
    # no position at all: zeros
    b.table[:] = -1
    assert not attend(km, b, q, 0.1).any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new,page", [([1], 1), ([40, 1], 1), ([200, 90], 1), ([1] * 12, 8), ([90], 8)])
def test_scores_of_minus_infinity_behind_missing_pages(km, dtype, new, page):
    """Rows that end among the missing pages see nothing, those behind them only -inf."""
    b = Paged(75, dtype, 2, 1, 64, page, new, [320] * len(new), 0)
    q = queries(b)
    q[..., 0] = 1
    b.k[..., 0] = -np.inf
    b.table[:, :280 // page] = -1
    got = attend(km, b, q, 0.1)
    for s in range(b.n_seqs):
        at = np.arange(320 - new[s], 320)
        rows = got[int(b.offsets[s]):int(b.offsets[s + 1])]
        assert not rows[at < 280].any()
        assert np.isnan(rows[at >= 280]).all()
