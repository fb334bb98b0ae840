"""How exactly attention over the paged cache weighs its values: f16 results carry the rounding of the
output and what fp32 arithmetic adds, no rounding of the softmax weights to f16, and weights far
below the largest one are not lost in long sequences."""
import math

import numpy as np
import pytest

import einsummable_amd as ea
from serving_oracle import HALF, NP, TINY, U32, Paged, assert_within, attention64
from test_gpu_attention_nonfinite import attend, queries

pytestmark = pytest.mark.gpu

F16, F32 = ea.F16, ea.F32


def bounds(b, q, scale, want):
    """[tokens, heads, dim].  A weight is off by
    * what its score is off by, a relative error: a sum of d products and four roundings more
      (scale, reference, exponential, fade), each of at most 2^-24 of sum |q||k| scale;
    * 2^-22, the two f16 parts it is multiplied in: 2^-11 of what the first leaves, 2^-11 of the weight;
    * the additions in fp32 that it passes through: one in sixteen or fewer positions of a wavefront,
      and at most 96 partial results of lanes, wavefronts and cuts;
    and so is the sum they are divided by, which doubles all of it.  A part below f16's least normal
    number is off by 2^-25, where the largest weight is 2^7 or more: 2^-32 of that for each position.
    Then the result is rounded to its type, half a step of what it is by then."""
    out = np.zeros(want.shape)
    for s in range(b.n_seqs):
        for j in range(b.new[s]):
            i = int(b.offsets[s]) + j
            pos = np.arange(b.lens[s] - b.new[s] + j + 1)
            k = np.repeat(b.rows(b.k, s, pos).astype(np.float64), b.group, axis=1)
            v = np.repeat(b.rows(b.v, s, pos).astype(np.float64), b.group, axis=1)
            qi = q[i].astype(np.float64)
            sc = scale * np.einsum("hd,phd->hp", qi, k)
            mag = abs(scale) * np.einsum("hd,phd->hp", np.abs(qi), np.abs(k)).max(axis=1)
            p = np.exp(sc - sc.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            weight = np.einsum("hp,phd->hd", p, np.abs(v))
            eps = 2 * ((b.d + 4) * U32 * mag[:, None] + 2.0 ** -22 + (pos.size / 16 + 96) * U32)
            out[i] = weight * eps
            if b.dtype == F16:
                out[i] += 2.0 ** -32 * p.max(axis=1)[:, None] * np.abs(v).sum(axis=0)
    return out * (1 + HALF[b.dtype]) + HALF[b.dtype] * np.abs(want) + TINY[b.dtype]


def run(km, b, q, scale):
    want, _ = attention64(b, q, scale)
    got = attend(km, b, q, scale)
    assert_within(got, want[:b.used], bounds(b, q, scale, want)[:b.used], "attention")


# few and many rows, shared and own positions, one key to hundreds
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("heads,kv,dim,new,lens,shared", [
    (4, 4, 16, [1] * 30, list(range(1, 31)), 0),
    (8, 2, 64, [1] * 20, [40 + 3 * i for i in range(20)], 33),
    (8, 2, 64, [2, 1], [45, 300], 33),
    (8, 1, 64, [30, 12], [30, 12], 0),
    (4, 1, 128, [9] * 6, [70 + i for i in range(6)], 50),
    (2, 1, 200, [50], [90], 0)])
def test_weights_are_not_rounded_to_f16(km, dtype, heads, kv, dim, new, lens, shared):
    b = Paged(80, dtype, heads, kv, dim, 16, new, lens, shared, spread=0.5)
    run(km, b, queries(b), dim ** -0.5)


def repeated(b, n):
    """The one sequence of b n times, over the same pages."""
    b.new, b.lens, b.n_seqs, b.tokens, b.used = b.new * n, b.lens * n, n, b.tokens * n, b.used * n
    b.offsets = np.concatenate([[0], np.cumsum(b.new)]).astype(np.int32)
    b.table = np.ascontiguousarray(np.repeat(b.table, n, axis=0))
    return b


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new,times,shared", [
    (1, 1, 0), (70, 1, 0),
    # as many sequences as leave each of them, or the prefix, in one part
    (1, 4100, 0), (70, 2100, 0), (1, 33000, 19999)])
@pytest.mark.parametrize("below", [20, 26, 28])
def test_small_weights_of_a_long_sequence_add_up(km, dtype, new, times, shared, below):
    """20000 positions of 2^-20 to 2^-28 of the first one's weight, and values of 1000 there."""
    b = Paged(81, dtype, 1, 1, 8, 256, [new], [20000], shared)
    b.k[..., 0] = -below
    b.v[:] = 1000
    b.k[b.table[0, 0], 0, :, 0] = 0
    b.v[b.table[0, 0], 0] = 0
    q = np.zeros((new, 1, 8), NP[dtype])
    q[..., 0] = 1
    want, _ = attention64(b, q, math.log(2))
    bound = bounds(b, q, math.log(2), want)
    got = attend(km, repeated(b, times), np.tile(q, (times, 1, 1)), math.log(2))
    assert_within(got, np.tile(want, (times, 1, 1)), np.tile(bound, (times, 1, 1)), "attention")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("new", [[1], [1] * 40, [80], [10] * 8])
def test_scores_that_rise_without_a_new_reference(km, dtype, new):
    """Scores that climb by less than 2^8 from the first step's, the largest values f16 has."""
    b = Paged(82, dtype, 2, 1, 64, 16, new, [400] * len(new), 0)
    q = np.zeros((b.tokens, 2, 64), NP[dtype])
    q[..., 0] = 1
    b.v[:] = 65504
    b.v[..., ::2] = 60000
    for s in range(b.n_seqs):
        for pos in range(400):
            b.k[b.table[s, pos // 16], pos % 16, :, 0] = pos / 400 * 7.99
    run(km, b, q, math.log(2))
