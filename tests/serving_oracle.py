"""Plain implementations in 64 bits of the serving operators, a builder of paged batches, and the
error bounds that the tests hold the kernels to.

A rounding to nearest is off by at most half a step of its type: 2^-11 of the value in f16 (and
2^-25 near zero), 2^-24 in f32.  A sum of n terms whose partial sums pass through at most `depth`
fp32 additions is off by at most depth * 2^-24 * sum |terms|.
"""
import numpy as np

import einsummable_amd as ea

NP = {ea.F16: np.float16, ea.F32: np.float32}
HALF = {ea.F16: 2.0 ** -11, ea.F32: 2.0 ** -24}
TINY = {ea.F16: 2.0 ** -25, ea.F32: 2.0 ** -149}
U32 = 2.0 ** -24


class Paged:
    """A batch over a paged cache: host arrays, and where every (sequence, position) lies."""

    def __init__(self, seed, dtype, heads, kv_heads, dim, page, new, lens, shared=0, tokens=None,
                 head_major=False, extra_cols=1, spread=1.0):
        r = np.random.RandomState(seed)
        self.r, self.dtype, self.page, self.shared = r, dtype, page, shared
        self.heads, self.kv, self.d, self.group = heads, kv_heads, dim, heads // kv_heads
        self.new, self.lens = list(new), list(lens)
        self.n_seqs = len(new)
        self.used = sum(new)
        self.tokens = self.used if tokens is None else tokens
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        cols = max(1, max(-(-max(ln, shared) // page) for ln in lens)) + extra_cols
        common = shared // page
        owned = [max(0, -(-max(ln, shared) // page) - common) for ln in lens]
        self.n_pages = common + sum(owned) + 2
        ids = r.permutation(self.n_pages)
        self.table = np.full((self.n_seqs, cols), -1, np.int32)
        at = common
        for s in range(self.n_seqs):
            self.table[s, :common] = ids[:common]
            self.table[s, common:common + owned[s]] = ids[at:at + owned[s]]
            at += owned[s]
        self.free = ids[at:]
        self.head_major = head_major
        shape = ((self.n_pages, kv_heads, page, dim) if head_major
                 else (self.n_pages, page, kv_heads, dim))
        self.k = (r.normal(0, spread, shape)).astype(NP[dtype])
        self.v = (r.normal(0, 1, shape)).astype(NP[dtype])
        tail = shared - common * page
        if tail:
            first = self.table[0, common]
            for s in range(1, self.n_seqs):
                for c in (self.k, self.v):
                    if head_major:
                        c[self.table[s, common], :, :tail] = c[first, :, :tail]
                    else:
                        c[self.table[s, common], :tail] = c[first, :tail]

    def strides(self):
        if self.head_major:
            return (self.kv * self.page * self.d, self.d, self.page * self.d)
        return (self.page * self.kv * self.d, self.kv * self.d, self.d)

    def rows(self, cache, s, positions):
        """[positions, kv heads, dim] of sequence s."""
        positions = np.asarray(positions, np.int64)
        pg, rw = self.table[s][positions // self.page], positions % self.page
        return cache[pg, :, rw] if self.head_major else cache[pg, rw]


def rotate64(x, freqs, rope):
    """x [n, heads, d], freqs [n, d/2, 2] -> float64"""
    x, f = x.astype(np.float64), freqs.astype(np.float64)
    if rope == ea.ROPE_NONE:
        return x
    h = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if rope == ea.ROPE_PAIRS else (x[..., :h], x[..., h:])
    c, s = f[:, None, :, 0], f[:, None, :, 1]
    y = np.empty_like(x)
    re, im = a * c - b * s, a * s + b * c
    if rope == ea.ROPE_PAIRS:
        y[..., 0::2], y[..., 1::2] = re, im
    else:
        y[..., :h], y[..., h:] = re, im
    return y


def rotate_bound(x, want, dtype, rope):
    """Two products and a sum in fp32 (three roundings of at most |a| + |b|, the factors being at
    most one), then the rounding to the type."""
    if rope == ea.ROPE_NONE:
        return np.zeros_like(want)
    x = np.abs(x.astype(np.float64))
    h = x.shape[-1] // 2
    if rope == ea.ROPE_PAIRS:
        both = np.repeat(x[..., 0::2] + x[..., 1::2], 2, axis=-1)
    else:
        both = np.concatenate([x[..., :h] + x[..., h:]] * 2, axis=-1)
    return 3 * U32 * both + HALF[dtype] * np.abs(want) * (1 + 2.0 ** -10) + TINY[dtype]


def attention64(b, q, scale, limit_of=None):
    """(out, bound), [tokens, heads, dim]; rows of no sequence are NaN in both."""
    out = np.full((b.tokens, b.heads, b.d), np.nan)
    bound = np.full_like(out, np.nan)
    for s in range(b.n_seqs):
        n, ln = b.new[s], b.lens[s]
        for j in range(n):
            i = int(b.offsets[s]) + j
            last = ln - n + j
            pos = np.arange(max(0, min(last + 1, b.table.shape[1] * b.page)))
            pages = b.table[s][pos // b.page]
            pos = pos[(pages >= 0) & (pages < b.n_pages)]
            if pos.size == 0:
                out[i], bound[i] = 0, 0
                continue
            k = np.repeat(b.rows(b.k, s, pos).astype(np.float64), b.group, axis=1)
            v = np.repeat(b.rows(b.v, s, pos).astype(np.float64), b.group, axis=1)
            qi = q[i].astype(np.float64)
            sc = scale * np.einsum("hd,phd->hp", qi, k)
            mag = abs(scale) * np.einsum("hd,phd->hp", np.abs(qi), np.abs(k)).max(axis=1)
            p = np.exp(sc - sc.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            out[i] = np.einsum("hp,phd->hd", p, v)
            weight = np.einsum("hp,phd->hd", p, np.abs(v))
            # scores: d products summed, scaled, and the reference subtracted, in fp32; the
            # exponential turns that absolute error into a relative one of p (and of the sum, so
            # twice), to which its own two steps, the fades of a wavefront's steps and the
            # additions of at most pos / 64 + 64 partial sums come
            eps = ((b.d + 8) * U32 * mag[:, None] +
                   (pos.size / 16 + 96) * 2 * U32) * 2
            bound[i] = weight * eps + HALF[b.dtype] * np.abs(out[i]) * 1.01 + TINY[b.dtype]
            if b.dtype == ea.F16:
                # p is rounded to f16 before the second product: 2^-11 of it, or 2^-25 of the
                # largest p where it is tiny
                bound[i] += weight * 2.0 ** -11 + 2.0 ** -25 * np.abs(v).sum(axis=0) * \
                    p.max(axis=1)[:, None]
    return out, bound


def int4_pack(q):
    """[n, k] integers 0..15 -> [n, k/2] bytes, the lower nibble the even k."""
    q = q.astype(np.uint8)
    return np.ascontiguousarray(q[:, 0::2] | (q[:, 1::2] << 4))


def int4_64(q, scales, zeros, x, group, dtype):
    """(y, bound): products are exact; a group's 128 (or fewer) products are summed by four
    matrix instructions, a wavefront adds at most k / 1024 such sums and eight or sixteen are joined."""
    of = np.arange(q.shape[1]) // group
    z = 8.0 if zeros is None else zeros.astype(np.float64)[:, of]
    w = (q.astype(np.float64) - z) * scales.astype(np.float64)[:, of]
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore"):   # rows of x may hold infinities and NaN
        y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    depth = 128 + q.shape[1] / 1024 + 16
    extra = 3 if dtype == ea.F32 else 0   # three parts: joining them, and 2^-33 of x left out
    return y, (depth + extra) * U32 * mag + HALF[dtype] * np.abs(y) * 1.01 + TINY[dtype]


def assert_within(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound)
    if bad.any():
        i = np.unravel_index(int(np.argmax(np.where(bad, np.abs(got - want) / (bound + 1e-300), 0))),
                             got.shape)
        raise AssertionError("%s: %d of %d values outside their bound; worst at %s: got %r want %r "
                             "(bound %g)" % (what, int(bad.sum()), got.size, i, got[i], want[i],
                                             bound[i]))
