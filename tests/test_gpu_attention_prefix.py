"""Attention over a shared prefix where not every sequence maps it: idle sequences, whose rows of the
page table hold anything, and sequences that end inside the prefix."""
import numpy as np
import pytest

import einsummable_amd as ea
from serving_oracle import Paged, assert_within, attention64
from test_gpu_attention_nonfinite import attend, queries

pytestmark = pytest.mark.gpu

F16, F32 = ea.F16, ea.F32


def check(km, b, fill):
    """`fill`: what the table holds behind a sequence's length, and all of an idle one's row."""
    for s in range(b.n_seqs):
        b.table[s, -(-b.lens[s] // b.page) if b.new[s] else 0:] = fill
    for s in range(b.n_seqs):
        if not b.new[s]:
            b.lens[s] = 1 << 20   # of a sequence long gone
    q = queries(b)
    want, bound = attention64(b, q, 0.1)
    got = attend(km, b, q, 0.1)
    assert_within(got, want[:b.used], bound[:b.used], "attention")


def batch(dtype, new, lens, shared, heads=4, kv=2, dim=64, page=8):
    return Paged(90, dtype, heads, kv, dim, page, new, lens, shared)


# what the first sequences are; behind them some that map the prefix, so many that its tiles have 16
# rows, 64 and 128
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("fill", [-1, "foreign"])
@pytest.mark.parametrize("more", [2, 20, 60])
@pytest.mark.parametrize("new,lens", [
    ([0], [1]), ([1], [24]), ([0, 0, 2], [1, 1, 40]), ([1, 0, 1, 3], [64, 1, 8, 95])])
def test_first_sequences_do_not_map_the_prefix(km, dtype, fill, more, new, lens):
    shared = 96
    b = batch(dtype, new + [1] * more, lens + [shared + 1 + 7 * i for i in range(more)], shared)
    check(km, b, int(b.free[0]) if fill == "foreign" else fill)


@pytest.mark.parametrize("n_idle", [63, 64, 300, 1500])
def test_many_idle_sequences_first(km, n_idle):
    new, lens = [0] * n_idle + [1, 2, 1], [1] * n_idle + [50, 130, 101]
    check(km, batch(F16, new, lens, 100), -1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("times", [1, 30])
def test_every_sequence_ends_inside_the_prefix(km, dtype, times):
    check(km, batch(dtype, [1, 0, 1, 2] * times, [20, 1, 45, 33] * times, 96), -1)
    # among more than a wavefront's lanes, the longest of all in the middle
    lens = [10 + i % 30 for i in range(150)]
    lens[97] = 77
    check(km, batch(dtype, [1] * 150, lens, 96), -1)


def test_page_table_shorter_than_the_prefix(km):
    b = batch(F16, [0, 1, 1], [1, 130, 150], 120)
    b.table = np.ascontiguousarray(b.table[:, :12])
    b.table[0] = -1
    q = queries(b)
    want, bound = attention64(b, q, 0.1)
    assert_within(attend(km, b, q, 0.1), want[:2], bound[:2], "attention")
