"""The serving operators (es_km_kv_append, es_km_prefix_attention, es_km_int4_linear) against
plain 64-bit implementations, at the sizes, masks and layouts where they can go wrong."""
import math

import numpy as np
import pytest

import einsummable_amd as ea
from einsummable_amd.llama_layer import freqs_cis_table
from helpers import assert_bits_equal, stream_handle
from serving_oracle import (NP, Paged, assert_within, attention64, int4_64, int4_pack, rotate64,
                            rotate_bound)

pytestmark = pytest.mark.gpu

F16, F32 = ea.F16, ea.F32
PAIRS, HALVES, NONE = ea.ROPE_PAIRS, ea.ROPE_HALVES, ea.ROPE_NONE


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class OnDevice:
    """The device arrays and descriptors of a Paged batch."""

    def __init__(self, b):
        self.k, self.v = dev(b.k), dev(b.v)
        self.offsets, self.lens = dev(b.offsets), dev(np.asarray(b.lens, np.int32))
        self.table = dev(b.table)
        self.cache = ea.KvCache(b.dtype, b.heads, b.kv, b.d, b.n_pages, b.page, self.k.data_ptr(),
                                self.v.data_ptr(), b.strides())
        self.batch = ea.KvBatch(b.n_seqs, b.tokens, self.offsets.data_ptr(), self.lens.data_ptr(),
                                self.table.data_ptr(), b.table.shape[1])


# ------------------------------------------------------------------------------ append

def expected_append(b, q, k, v, freqs, rope, q_before):
    """(q_out, its bound, k cache, its bound, v cache)."""
    qo, qb = q_before.astype(np.float64), np.zeros(q_before.shape)
    kc, vc = b.k.astype(np.float64), b.v.copy()
    kb = np.zeros(kc.shape)
    for s in range(b.n_seqs):
        for j in range(b.new[s]):
            i = int(b.offsets[s]) + j
            pos = b.lens[s] - b.new[s] + j
            if pos < 0 or (rope != NONE and pos >= freqs.shape[0]):
                continue
            f = freqs[pos:pos + 1] if rope != NONE else None
            qo[i] = rotate64(q[i:i + 1], f if f is not None else q[:1], rope)[0]
            qb[i] = rotate_bound(q[i:i + 1], qo[i:i + 1], b.dtype, rope)[0]
            col = pos // b.page
            page = b.table[s, col] if col < b.table.shape[1] else -1
            if page < 0 or page >= b.n_pages:
                continue
            at = (page, slice(None), pos % b.page) if b.head_major else (page, pos % b.page)
            kc[at] = rotate64(k[i:i + 1], f if f is not None else q[:1], rope)[0]
            kb[at] = rotate_bound(k[i:i + 1], kc[at][None], b.dtype, rope)[0]
            vc[at] = v[i]
    return qo, qb, kc, kb, vc


def run_append(km, b, rope, n_pos=None, packed=False, in_place=False, with_q=True):
    import torch

    dt = NP[b.dtype]
    qkv = b.r.normal(0, 1, (b.tokens, b.heads + 2 * b.kv, b.d)).astype(dt)
    q, k, v = (np.ascontiguousarray(x) for x in
               (qkv[:, :b.heads], qkv[:, b.heads:b.heads + b.kv], qkv[:, b.heads + b.kv:]))
    n_pos = n_pos or max(max(b.lens), 1)
    freqs = freqs_cis_table(n_pos, b.d // 2)
    g = OnDevice(b)
    e = np.dtype(dt).itemsize
    if packed:
        d_qkv = dev(qkv)
        p = d_qkv.data_ptr()
        ptrs = (p, p + b.heads * b.d * e, p + (b.heads + b.kv) * b.d * e)
        st = (b.heads + 2 * b.kv) * b.d
        strides = (st, st, st)
    else:
        d_q, d_k, d_v = dev(q), dev(k), dev(v)
        ptrs = (d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr())
        strides = (b.heads * b.d, b.kv * b.d, b.kv * b.d)
    before = b.r.normal(0, 1, q.shape).astype(dt)
    if in_place:
        assert not packed
        d_out, before, out_stride = d_q, q, strides[0]
    else:
        # rows further apart than they are wide
        out_stride = b.heads * b.d + 16
        wide = np.zeros((b.tokens, out_stride), dt)
        wide[:, :b.heads * b.d] = before.reshape(b.tokens, -1)
        d_out = dev(wide)
    d_f = dev(freqs)
    km.kv_append(g.cache, g.batch, stream_handle(), d_out.data_ptr() if with_q else 0,
                 ptrs[0] if with_q else 0, ptrs[1], ptrs[2], rope,
                 d_f.data_ptr() if rope != NONE else 0, n_pos if rope != NONE else 0,
                 (out_stride,) + strides)
    torch.cuda.synchronize()
    qo, qb, kc, kb, vc = expected_append(b, q, k, v, freqs, rope, before)
    got = d_out.cpu().numpy().reshape(b.tokens, -1)
    if not in_place:
        assert not got[:, b.heads * b.d:].any()
    if with_q:
        assert_within(got[:, :b.heads * b.d].reshape(q.shape), qo, qb, "q_out")
    else:
        assert_bits_equal(got[:, :b.heads * b.d].reshape(q.shape), before, "q_out")
    # bounds are zero, hence equality, wherever nothing was to be written
    assert_within(g.k.cpu().numpy(), kc, kb, "k cache")
    assert_bits_equal(g.v.cpu().numpy(), vc, "v cache")


@pytest.mark.parametrize("rope", [PAIRS, HALVES, NONE])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 128, 16), (6, 2, 64, 5), (5, 1, 8, 1),
                                               (3, 3, 40, 24), (2, 1, 256, 64)])
def test_append(km, rope, dtype, heads, kv, dim, page):
    b = Paged(1, dtype, heads, kv, dim, page, new=[1, 0, 7, 1, 0, 33], lens=[1, 5, 70, 17, 0, 33])
    run_append(km, b, rope)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_packed_projection_and_in_place(km, dtype):
    new, lens = [3, 1, 9], [30, 1, 9]
    run_append(km, Paged(2, dtype, 8, 2, 64, 16, new, lens), HALVES, packed=True)
    run_append(km, Paged(3, dtype, 8, 2, 64, 16, new, lens, head_major=True), PAIRS, packed=True)
    run_append(km, Paged(4, dtype, 8, 2, 64, 16, new, lens), PAIRS, in_place=True)
    run_append(km, Paged(5, dtype, 8, 2, 64, 16, new, lens), HALVES, in_place=True)
    run_append(km, Paged(6, dtype, 8, 2, 64, 16, new, lens), HALVES, with_q=False)


def test_append_drops_what_has_no_place(km):
    # rows behind the last sequence, tokens before position 0, beyond the table of frequencies,
    # on pages that do not exist or have no column
    b = Paged(7, F16, 4, 2, 64, 8, new=[2, 5, 3, 1], lens=[40, 3, 20, 9], tokens=15)
    b.table[2, 2] = -1
    b.table[3, 1] = b.n_pages
    run_append(km, b, PAIRS, n_pos=39)
    b = Paged(8, F16, 4, 2, 64, 8, new=[4], lens=[34], extra_cols=0)
    b.table = np.ascontiguousarray(b.table[:, :4])
    run_append(km, b, HALVES)


@pytest.mark.parametrize("n_seqs", [64, 65, 700, 5000])
def test_append_many_sequences(km, n_seqs):
    r = np.random.RandomState(n_seqs)
    new = [int(x) for x in r.choice([0, 0, 1, 1, 1, 2], n_seqs)]
    lens = [n + int(x) for n, x in zip(new, r.randint(0, 9, n_seqs))]
    run_append(km, Paged(9, F16, 2, 1, 16, 4, new, lens), PAIRS)


def test_append_prompt(km):
    # enough tokens for the form that takes several heads per thread
    run_append(km, Paged(10, F16, 9, 3, 80, 16, [600, 1, 130], [640, 90, 130]), PAIRS)
    run_append(km, Paged(11, F32, 32, 32, 64, 32, [513], [600]), HALVES)


# ------------------------------------------------------------------------------ attention

def run_attention(km, b, scale=None, spread=1.0, shared=None, check=True, stream=None):
    import torch

    dt = NP[b.dtype]
    scale = 1.0 / math.sqrt(b.d) if scale is None else scale
    q = b.r.normal(0, spread, (b.tokens, b.heads, b.d)).astype(dt)
    g = OnDevice(b)
    shared = b.shared if shared is None else shared
    need = km.prefix_attention_workspace(g.cache, b.n_seqs, b.tokens, shared)
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")   # NaN everywhere
    st_q, st_o = b.heads * b.d + 8, b.heads * b.d + 16
    wide = np.zeros((b.tokens, st_q), dt)
    wide[:, :b.heads * b.d] = q.reshape(b.tokens, -1)
    d_q = dev(wide)
    before = b.r.normal(0, 1, (b.tokens, st_o)).astype(dt)
    d_o = dev(before)
    torch.cuda.synchronize()
    km.prefix_attention(g.cache, g.batch, shared, scale,
                        stream_handle() if stream is None else stream, d_o.data_ptr(),
                        d_q.data_ptr(), (ws.data_ptr(), need) if need else None, (st_o, st_q))
    torch.cuda.synchronize()
    got = d_o.cpu().numpy()
    assert_bits_equal(got[:, b.heads * b.d:], before[:, b.heads * b.d:], "between the rows")
    used = int(b.offsets[-1])
    assert_bits_equal(got[used:], before[used:], "rows behind the last sequence")
    got = got[:used, :b.heads * b.d].reshape(used, b.heads, b.d)
    if check:
        want, bound = attention64(b, q, scale)
        assert_within(got, want[:used], bound[:used], "attention")
    return got


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,dim,page,shared", [
    (4, 4, 128, 16, 0), (4, 4, 128, 16, 100), (8, 2, 64, 5, 33), (6, 2, 64, 24, 1),
    (32, 1, 64, 1, 7), (3, 3, 40, 24, 64), (2, 1, 256, 64, 130), (5, 1, 200, 16, 31),
    (4, 1, 8, 7, 32)])
def test_attention(km, dtype, heads, kv, dim, page, shared):
    b = Paged(20, dtype, heads, kv, dim, page, [1, 0, 1, 3, 17, 1],
              [shared + own for own in (1, 9, 70, 3, 40, 200)], shared)
    run_attention(km, b)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_lengths_of_zero_and_one_and_shorter_than_the_prefix(km, dtype):
    # a token at position 0, sequences that end inside the prefix, one whose length is less than
    # its number of new tokens (the first of them see nothing), an empty one
    b = Paged(21, dtype, 4, 2, 64, 16, [1, 2, 1, 5, 3, 0], [1, 20, 0, 3, 90, 0], shared=48,
              tokens=14)
    run_attention(km, b)
    b = Paged(22, dtype, 4, 2, 64, 16, [1, 1], [1, 0], shared=0)
    run_attention(km, b)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("shared", [0, 65])
@pytest.mark.parametrize("more", [0, 80])
def test_attention_ignores_what_masked_places_hold(km, dtype, shared, more):
    b = Paged(23, dtype, 4, 2, 64, 8, [6 + more, 1 + more, 20],
              [shared + 6 + more, shared + 19 + more, shared + 41], shared)
    clean = run_attention(km, b)
    for bad in (np.nan, np.inf, -np.inf):
        for which in (b.k, b.v):
            which[b.free] = bad                                  # pages of nobody
            for s, ln in enumerate(b.lens):
                for pos in range(ln, -(-ln // b.page) * b.page):  # behind the last position
                    which[b.table[s, pos // b.page], pos % b.page] = bad
    b.r = np.random.RandomState(23)   # the same queries again
    b2 = Paged(23, dtype, 4, 2, 64, 8, b.new, b.lens, shared)
    b.r = b2.r
    got = run_attention(km, b)
    assert_bits_equal(got, clean, "what lies behind the sequences")
    # a token's own values that are not finite reach the rows that see it, and no others
    b3 = Paged(23, dtype, 4, 2, 64, 8, b.new, b.lens, shared)
    s, at = 2, b.lens[2] - 5                       # token 15 of 20 of the third sequence
    where = (b3.table[s, at // 8], at % 8)
    b3.v[where][:, 3] = np.inf
    b3.v[where][:, 4] = np.nan
    got = run_attention(km, b3, check=False)
    first = int(b3.offsets[2]) + 15
    assert_bits_equal(got[:first], clean[:first], "rows before the token")
    assert np.isposinf(got[first:, :, 3]).all() and np.isnan(got[first:, :, 4]).all()
    keep = [i for i in range(64) if i not in (3, 4)]
    assert_bits_equal(got[:, :, keep], clean[:, :, keep], "other elements")


def test_attention_leaves_out_pages_that_do_not_exist(km):
    b = Paged(24, F16, 4, 2, 64, 8, [1, 4, 1], [50, 61, 33])
    b.table[0, 2] = -1
    b.table[1, 7] = b.n_pages        # the page of the newest tokens
    b.table[2, :] = 1 << 30          # none at all: zeros
    got = run_attention(km, b)
    assert not got[5].any()
    # the same with tiles of many rows, in shared and in own positions
    b = Paged(33, F16, 4, 2, 64, 8, [40, 1, 70], [140, 101, 190], shared=70)
    b.table[:, 3] = -1
    b.table[0, 12] = b.n_pages
    b.table[2, 9:] = -7
    run_attention(km, b)
    b = Paged(34, F16, 4, 2, 128, 8, [1] * 40, [90] * 40, shared=70)
    b.table[:, 5] = -1
    b.table[7, 10] = -1
    run_attention(km, b)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_attention_scale_of_zero_and_below(km, dtype, scale):
    run_attention(km, Paged(35, dtype, 4, 2, 64, 8, [1, 3], [70, 33], shared=20), scale=scale)
    run_attention(km, Paged(36, dtype, 4, 2, 64, 8, [50, 3], [70, 33], shared=20), scale=scale)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_is_the_same_whatever_part_is_called_shared(km, dtype):
    base = None
    for shared in (0, 1, 40, 63, 64):
        b = Paged(25, dtype, 8, 2, 64, 16, [1, 1, 2, 1], [65, 100, 130, 64 + 77], shared=64)
        got = run_attention(km, b, shared=shared).astype(np.float64)
        base = got if base is None else base
        # two results within their bounds of the same value
        np.testing.assert_allclose(got, base, atol=4e-3 if dtype == F16 else 1e-5)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("spread", [0.01, 30.0])
def test_attention_flat_and_peaked_scores(km, dtype, spread):
    b = Paged(26, dtype, 4, 2, 128, 16, [1, 3, 1], [400, 300, 77], shared=50, spread=spread)
    run_attention(km, b, spread=1.0)


def test_attention_long_and_many(km):
    # one long sequence beside short ones: its positions are cut finer than theirs
    run_attention(km, Paged(27, F16, 4, 1, 64, 16, [1] * 8, [9000] + [20] * 7))
    # a single sequence, nothing shared
    run_attention(km, Paged(28, F16, 8, 8, 128, 16, [1], [3001]))
    # more sequences than threads
    r = np.random.RandomState(5)
    new = [int(x) for x in r.choice([0, 1, 1, 2], 700)]
    run_attention(km, Paged(29, F16, 2, 1, 64, 16, new, [n + 40 + i % 50 for i, n in
                                                         enumerate(new)], shared=40))
    # a prompt: no cuts, causal tiles
    run_attention(km, Paged(30, F16, 4, 2, 64, 16, [190, 3], [190, 200]))


def test_attention_head_major_pages(km):
    run_attention(km, Paged(31, F16, 8, 4, 128, 16, [1, 2], [70, 55], shared=33, head_major=True))


def test_attention_is_deterministic_and_runs_on_other_streams(km):
    import torch

    def make():
        return Paged(32, F16, 8, 2, 128, 16, [1] * 20, [300 + 37 * i for i in range(20)],
                     shared=256)
    first = run_attention(km, make(), check=False)
    side = torch.cuda.Stream()
    for _ in range(3):
        assert_bits_equal(run_attention(km, make(), check=False, stream=side.cuda_stream), first,
                          "repeated")


# ------------------------------------------------------------------------------ int4

def run_int4(km, seed, dtype, m, k, n, group, zeros=None, pad=0, x=None, spread=1.0):
    import torch

    r = np.random.RandomState(seed)
    dt = NP[dtype]
    groups = -(-k // group)
    q = r.randint(0, 16, (n, k))
    scales = (0.01 * r.uniform(0.5, 2, (n, groups))).astype(dt)
    z = None
    if zeros is not None:
        z = r.randint(zeros[0], zeros[1] + 1, (n, groups)).astype(np.uint8)
    if x is None:
        x = r.normal(0, spread, (m, k)).astype(dt)
    w = np.zeros((n, k // 2 + pad * 16), np.uint8)
    w[:, :k // 2] = int4_pack(q)
    sp = np.zeros((n, groups + pad), dt)
    sp[:, :groups] = scales
    zp = np.zeros((n, groups + pad), np.uint8)
    if z is not None:
        zp[:, :groups] = z
    xp = np.zeros((m, k + 8 * pad), dt)
    xp[:, :k] = x
    d_w, d_s, d_z, d_x = dev(w), dev(sp), dev(zp), dev(xp)
    y0 = r.normal(0, 1, (m, n + 3 * pad)).astype(dt)
    d_y = dev(y0)
    wt = ea.Int4Weight(dtype, n, k, group, d_w.data_ptr(), d_s.data_ptr(),
                       d_z.data_ptr() if z is not None else 0, w.shape[1], groups + pad)
    need = km.int4_linear_workspace(wt, m)
    assert (need > 0) == (dtype == F32)
    ws = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    km.int4_linear(wt, m, stream_handle(), d_y.data_ptr(), d_x.data_ptr(),
                   (ws.data_ptr(), need) if need else None, (n + 3 * pad, k + 8 * pad))
    torch.cuda.synchronize()
    got = d_y.cpu().numpy()
    assert_bits_equal(got[:, n:], y0[:, n:], "between the rows")
    want, bound = int4_64(q, scales, z, x, group, dtype)
    return got[:, :n], want, bound


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("m,k,n,group", [
    (1, 32, 1, 32), (1, 4096, 250, 128), (2, 96, 17, 32), (5, 160, 33, 64), (6, 1056, 15, 96),
    (16, 2048, 48, 256), (17, 512, 16, 32), (21, 288, 40, 288), (33, 1184, 31, 128),
    (70, 256, 64, 4096), (3, 11008, 20, 32), (64, 640, 18, 160)])
def test_int4(km, dtype, m, k, n, group):
    got, want, bound = run_int4(km, 40, dtype, m, k, n, group)
    assert_within(got, want, bound, "int4")
    got, want, bound = run_int4(km, 41, dtype, m, k, n, group, zeros=(0, 15), pad=1)
    assert_within(got, want, bound, "int4 with zero points")


@pytest.mark.parametrize("dtype", [F16, F32])
def test_int4_zero_points_beyond_the_nibble(km, dtype):
    got, want, bound = run_int4(km, 42, dtype, 3, 512, 40, 64, zeros=(0, 255))
    assert_within(got, want, bound, "int4, zero points up to 255")


@pytest.mark.parametrize("scale", [1e-42, 1e-30, 1.0, 1e30])
def test_int4_f32_range_of_a_row(km, scale):
    # rows that span 2^20 in magnitude, at both ends of what f32 holds
    r = np.random.RandomState(43)
    x = (r.normal(0, 1, (4, 640)) * 2.0 ** r.randint(-20, 1, (4, 640)) * scale).astype(np.float32)
    x[2] = 0
    got, want, bound = run_int4(km, 44, F32, 4, 640, 33, 64, x=x)
    assert_within(got, want, bound, "int4 f32 range")
    assert not got[2].any()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_int4_rows_do_not_touch_each_other(km, dtype):
    r = np.random.RandomState(45)
    x = r.normal(0, 1, (6, 320)).astype(NP[dtype])
    clean, want, bound = run_int4(km, 46, dtype, 6, 320, 24, 64, x=x)
    x[1, 5], x[4, 7], x[4, 9] = np.inf, np.nan, -np.inf
    got, _, _ = run_int4(km, 46, dtype, 6, 320, 24, 64, x=x)
    for i in (0, 2, 3, 5):
        assert_bits_equal(got[i], clean[i], "row %d" % i)
    assert not np.isfinite(got[1]).any() and np.isnan(got[4]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("m,k,n,group", [
    (1, 160, 16390, 32), (2, 224, 16384, 64), (4, 160, 16417, 96), (8, 256, 16400, 128),
    (12, 96, 16391, 64), (24, 160, 8205, 32), (64, 128, 16385, 128), (67, 160, 8200, 160)])
def test_int4_many_columns(km, dtype, m, k, n, group):
    got, want, bound = run_int4(km, 47, dtype, m, k, n, group, zeros=(0, 15), pad=1)
    assert_within(got, want, bound, "int4, many columns")


# ------------------------------------------------------------------------------ streams, sizes

def test_attention_many_rows_of_many_sequences(km):
    """Tiles of 64 and 128 rows with more sequences than lanes, and than threads."""
    for n_seqs, heads, most in ((70, 16, 5), (300, 32, 6)):
        r = np.random.RandomState(n_seqs)
        new = [int(x) for x in r.randint(0, most + 1, n_seqs)]
        lens = [n + int(x) for n, x in zip(new, r.randint(0, 90, n_seqs))]
        run_attention(km, Paged(33, F16, heads, 1, 64, 16, new, lens))


def test_cache_offsets_beyond_32_bits(km):
    """Pages 3 GiB apart: entries of the last pages lie behind 2^32 elements.  The bytes of a
    compact cache."""
    import torch

    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    b = Paged(34, F16, 8, 2, 128, 16, [1, 4, 1], [60, 37, 20], shared=17)
    b.n_pages = b.k.shape[0]
    assert b.n_pages <= 12
    page = 16 * 2 * 128
    far = 3 << 29
    assert (b.n_pages - 1) * far > 1 << 32
    near = OnDevice(b)
    q = dev(b.r.normal(0, 1, (6, 8, 128)).astype(np.float16))
    k = dev(b.r.normal(0, 1, (6, 2, 128)).astype(np.float16))
    wide = torch.empty((b.n_pages - 1) * far + page, dtype=torch.float16, device="cuda")
    pages = [wide[p * far:p * far + page].view(16, 2, 128) for p in range(b.n_pages)]
    outs = []
    for base, stride in ((near.k, page), (wide, far)):
        if base is wide:
            fresh = OnDevice(b)
            for p in range(b.n_pages):
                pages[p].copy_(fresh.k[p])
        cache = ea.KvCache(F16, 8, 2, 128, b.n_pages, 16, base.data_ptr(), base.data_ptr(),
                           (stride, 256, 128))
        # keys and values share the buffer: a value written last is read as both
        km.kv_append(cache, near.batch, stream_handle(), 0, 0, k.data_ptr(), k.data_ptr(), NONE)
        need = km.prefix_attention_workspace(cache, 3, 6, 17)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(q)
        km.prefix_attention(cache, near.batch, 17, 0.09, stream_handle(), out.data_ptr(),
                            q.data_ptr(), (ws.data_ptr(), need))
        torch.cuda.synchronize()
        outs.append(out.cpu().numpy())
    assert_bits_equal(outs[1], outs[0], "attention")
    for p in range(b.n_pages):
        assert_bits_equal(pages[p].cpu().numpy(), near.k[p].cpu().numpy(), "page %d" % p)
    assert outs[0].any()


def test_calls_at_once_on_two_streams(km):
    """Attention, append and int4 products in flight on two streams, a workspace each: the bytes
    of one after the other."""
    import torch

    def job(seed):
        b = Paged(seed, F16, 8, 2, 128, 16, [1, 2] * 10, [200 + 31 * i for i in range(20)],
                  shared=128)
        g = OnDevice(b)
        r = b.r
        q = dev(r.normal(0, 1, (30, 8, 128)).astype(np.float16))
        kv = dev(r.normal(0, 1, (30, 2, 128)).astype(np.float16))
        w = dev(r.randint(0, 256, (1024, 512)).astype(np.uint8))
        s = dev(r.uniform(0.01, 0.02, (1024, 8)).astype(np.float32))
        x = dev(r.normal(0, 1, (30, 1024)).astype(np.float32))
        wt = ea.Int4Weight(F32, 1024, 1024, 128, w.data_ptr(), s.data_ptr())
        need = (km.prefix_attention_workspace(g.cache, 20, 30, 128),
                km.int4_linear_workspace(wt, 30))
        ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in need]
        out, y = torch.zeros_like(q), torch.zeros(30, 1024, device="cuda")

        def go(stream):
            for _ in range(4):
                km.kv_append(g.cache, g.batch, stream, 0, 0, kv.data_ptr(), kv.data_ptr(), NONE)
                km.prefix_attention(g.cache, g.batch, 128, 0.1, stream, out.data_ptr(),
                                    q.data_ptr(), (ws[0].data_ptr(), need[0]))
                km.int4_linear(wt, 30, stream, y.data_ptr(), x.data_ptr(),
                               (ws[1].data_ptr(), need[1]))

        def take():
            got = out.cpu().numpy(), y.cpu().numpy(), g.k.cpu().numpy()
            out.zero_()
            y.zero_()
            return got
        go.keep = (g, q, kv, w, s, x, ws)
        return go, take

    jobs = [job(35), job(36)]
    want = []
    for go, take in jobs:
        go(stream_handle())
        torch.cuda.synchronize()
        want.append(take())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for (go, _), s in zip(jobs, streams):
        go(s.cuda_stream)
    torch.cuda.synchronize()
    for (_, take), first in zip(jobs, want):
        for a, c in zip(take(), first):
            assert_bits_equal(a, c, "two streams")
