"""The paged cache's operators and attention over packed rows, against the formulas in 64
bits (numpy), at the sizes and contents where they can go wrong: lengths of zero and one,
ends inside tiles and pages, NaN and infinities in every place that no row may see, pages
that are not there, padded batches, strides, and captured calls replayed on new contents."""
from __future__ import annotations

import numpy as np
import pytest

import mi_attn
from mi_attn import U32, AttentionConfig, QkNormRopeCacheConfig
from helpers import f16

pytestmark = pytest.mark.gpu
THETA, EPS = 1e6, 1e-6
HALF_STEP = 2.0 ** -11  # f16 rounding, relative
NOWHERE = 0xFFFFFFFF


def bits(a: np.ndarray) -> np.ndarray:
    return np.asarray(a, dtype=np.float64).astype(np.float16).view(np.uint16)


def poison(rng, shape) -> np.ndarray:
    """f16 NaN, infinities and the largest values."""
    return rng.choice(np.array([0x7E00, 0xFE00, 0x7C00, 0xFC00, 0x7BFF, 0xFBFF], np.uint16), shape)


def attend(q, k, v, seen, f16_weights):
    """Rows q [n, Hq, D] over k / v [L, Hkv, D]; seen[i] lists row i's keys. The result in 64
    bits, and how far a kernel's may be off, element by element:
     - its rounding to f16: half a step of the result (2^-25 below f16's smallest normal);
     - a score of D products summed in f32 is off by D 2^-24 sum |q k|, scaled, and its
       exponent's argument and 2^x by 2^-20 together; a weight is off by that much relative
       to itself, in the weighted sum and in the row sum; both sums of L terms by L 2^-24;
     - weights rounded to f16 (packed rows): half a step of each in both sums, and 2^-33 of
       the row's largest below f16's normal range (bias 2^8)."""
    n, hq, d = q.shape
    group = hq // k.shape[1]
    out, tol = np.full((n, hq, d), np.nan), np.zeros((n, hq, d))
    for i in range(n):
        keys = seen[i]
        if len(keys) == 0:
            continue
        kk, vv = k[keys].astype(np.float64), v[keys].astype(np.float64)
        for h in range(hq):
            a, b = kk[:, h // group], vv[:, h // group]
            s = a @ q[i, h] / np.sqrt(d)
            p = np.exp(s - s.max())
            total = p.sum()
            p /= total
            r = p @ b
            size = p @ np.abs(b)
            weight = d * 2.0 ** -24 * (np.abs(a) @ np.abs(q[i, h])).max() / np.sqrt(d) + 2.0 ** -20
            off = 2 * weight * size + 2 * len(keys) * 2.0 ** -24 * size
            if f16_weights:
                off = off + HALF_STEP * (size + np.abs(r)) + 2 * len(keys) * 2.0 ** -33 * np.abs(b).max(0) / total
            out[i, h], tol[i, h] = r, off + HALF_STEP * (np.abs(r) + off) + 2.0 ** -25
    return out, tol


def hold(got_bits, want, tol, label=""):
    got = f16(got_bits).astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{label}: NaN in other places"
    there = ~np.isnan(want)
    over = np.abs(got - want)[there] - np.broadcast_to(tol, want.shape)[there]
    assert over.size == 0 or over.max() <= 0, f"{label}: {over.max():.3e} past the tolerance"


class Cache:
    """A pool of pages with poison in every slot that no sequence has filled."""

    def __init__(self, ctx, rng, lengths, width, size, hkv, d, layout="head_major", extra=3, missing=()):
        self.ctx, self.size, self.hkv, self.d, self.layout = ctx, size, hkv, d, layout
        b = len(lengths)
        self.pages = b * width + extra
        order = rng.permutation(self.pages)
        self.table = order[:b * width].reshape(b, width).astype(np.uint32)
        self.lengths = np.asarray(lengths)
        for i, n in enumerate(lengths):  # the tail of a row names no page
            self.table[i, -(-int(n) // size):] = rng.choice([NOWHERE, self.pages, self.pages + 7])
        for i, page in missing:
            self.table[i, page] = NOWHERE
        self.rows = [(rng.standard_normal((n, hkv, d)).astype(np.float16),
                      rng.standard_normal((n, hkv, d)).astype(np.float16)) for n in lengths]
        self.key, self.value = (poison(rng, (self.pages, size, hkv, d)) for _ in "kv")
        for i, (k, v) in enumerate(self.rows):
            for p in range(len(k)):
                page = self.table[i, p // size]
                if page < self.pages:
                    self.key[page, p % size] = k[p].view(np.uint16)
                    self.value[page, p % size] = v[p].view(np.uint16)
        self.owners = []
        self.key_pages, self.value_pages = self.upload(self.key), self.upload(self.value)
        self.device_table = self.upload_table()
        self.device_lengths = ctx.tensor(np.asarray(lengths, np.uint32), U32)

    def upload(self, logical):
        """[P, S, H, D] rows as a view of the layout's storage."""
        p, s, h, d = logical.shape
        if self.layout == "position_major":
            owner = self.ctx.tensor(np.ascontiguousarray(logical))
            self.owners.append(owner)
            return owner
        if self.layout == "head_major":
            owner = self.ctx.tensor(np.ascontiguousarray(logical.transpose(0, 2, 1, 3)))
            self.owners.append(owner)
            return owner.view((p, s, h, d), (h * s * d, d, s * d, 1))
        # "gaps": padded rows, pages last to first.
        store = np.full((p, h, s, d + 8), 0x7E00, np.uint16)
        store[..., :d] = logical.transpose(0, 2, 1, 3)[::-1]
        owner = self.ctx.tensor(store)
        self.owners.append(owner)
        w = d + 8
        return owner.view((p, s, h, d), (-h * s * w, w, s * w, 1), offset=(p - 1) * h * s * w)

    def upload_table(self):
        b, m = self.table.shape
        store = np.full((b, m + 5), 12345678, np.uint32)
        store[:, :m] = self.table
        owner = self.ctx.tensor(store, U32)
        self.owners.append(owner)
        return owner.view((b, m), (m + 5, 1))

    def download(self, which):
        """[P, S, H, D] bits of a pool."""
        owner = self.owners[which]
        p, s, h, d = self.pages, self.size, self.hkv, self.d
        raw = self.ctx.download(owner)
        if self.layout == "position_major":
            return raw
        if self.layout == "head_major":
            return raw.transpose(0, 2, 1, 3)
        return raw[::-1, :, :, :d].transpose(0, 2, 1, 3)

    def there(self, i, upto):
        """Positions below `upto` of sequence i that have a page."""
        at = np.arange(upto)
        return at[self.table[i, at // self.size] < self.pages] if upto else at


def padded_rows(ctx, rows, pad=8):
    """Device rows [n, H, D] with a gap between rows: (owner, view)."""
    n, h, d = rows.shape
    store = np.full((n, h * d + pad), 0x7E00, np.uint16)
    store[:, :h * d] = rows.view(np.uint16).reshape(n, h * d)
    owner = ctx.tensor(store)
    return owner, owner.view((n, h, d), (h * d + pad, d, 1))


# ------------------------------------------------------------------- decode --

EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200]


def decode(ctx, cache, q, hq):
    cfg = AttentionConfig(hq, cache.hkv, cache.d, True, 77)
    owner, view = padded_rows(ctx, q)
    out = ctx.empty(q.shape)
    batch = ctx.begin_batch()
    batch.attention_decode_paged(view, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                                 cfg, out=out)
    batch.finish()
    return ctx.download(out)


def decode_want(cache, q):
    outs, tols = [], []
    for i in range(len(q)):
        k, v = cache.rows[i]
        want, tol = attend(q[i:i + 1].astype(np.float64), k, v, [cache.there(i, len(k))], False)
        outs.append(want[0])
        tols.append(tol[0])
    return np.array(outs), np.array(tols)


@pytest.mark.parametrize("hq,hkv,d,size,layout", [
    (8, 2, 128, 16, "head_major"), (8, 8, 64, 16, "position_major"), (5, 1, 256, 32, "gaps"), (12, 4, 32, 64, "gaps"),
    (20, 1, 128, 32, "position_major"), (7, 7, 128, 128, "head_major"), (48, 2, 64, 16, "gaps"),
    (16, 1, 32, 16, "position_major"), (40, 8, 128, 256, "position_major")])
def test_decode_at_the_edges_of_tiles_and_pages(ctx, hq, hkv, d, size, layout):
    rng = np.random.default_rng(hq * d + size)
    cache = Cache(ctx, rng, EDGES, -(-210 // size), size, hkv, d, layout)
    q = (1.5 * rng.standard_normal((len(EDGES), hq, d))).astype(np.float16)
    hold(decode(ctx, cache, q, hq), *decode_want(cache, q), f"decode {hq}/{hkv}/{d} page {size}")


@pytest.mark.parametrize("hq,hkv,d,size,lengths", [
    (8, 2, 128, 16, [5000]), (4, 2, 64, 64, [3001, 20, 1, 0, 777]), (2, 1, 256, 32, [1500, 1501]),
    (6, 2, 32, 16, [4097, 4096]), (16, 8, 128, 16, list(range(1, 150, 3)))])
def test_decode_longer_and_ragged(ctx, hq, hkv, d, size, lengths):
    rng = np.random.default_rng(d + size)
    cache = Cache(ctx, rng, lengths, -(-max(lengths) // size) + 1, size, hkv, d)
    q = (1.5 * rng.standard_normal((len(lengths), hq, d))).astype(np.float16)
    first = decode(ctx, cache, q, hq)
    hold(first, *decode_want(cache, q), f"decode {lengths[:3]}")
    assert np.array_equal(first, decode(ctx, cache, q, hq)), "two calls differ"


def test_decode_without_some_pages(ctx):
    """Keys of a page that is not there are not seen; a sequence without any is NaN."""
    rng = np.random.default_rng(5)
    missing = [(0, 0), (1, 1), (1, 4), (2, 2), (3, 0), (3, 1), (4, 12), (5, 3), (5, 4), (5, 5)]
    cache = Cache(ctx, rng, [40, 200, 47, 32, 200, 100], 13, 16, 2, 128, missing=missing)
    q = rng.standard_normal((6, 8, 128)).astype(np.float16)
    want, tol = decode_want(cache, q)
    assert np.isnan(want[3]).all()
    hold(decode(ctx, cache, q, 8), want, tol)


def test_decode_lengths_past_the_table_are_clamped(ctx):
    rng = np.random.default_rng(6)
    cache = Cache(ctx, rng, [64, 48], 4, 16, 2, 64)
    ctx.upload(cache.device_lengths, np.array([NOWHERE, 48], np.uint32))
    q = rng.standard_normal((2, 4, 64)).astype(np.float16)
    hold(decode(ctx, cache, q, 4), *decode_want(cache, q))


def test_decode_scores_far_apart_and_values_not_finite(ctx):
    """One key far above the rest, equal keys, and an infinity that a row does see."""
    rng = np.random.default_rng(7)
    cache = Cache(ctx, rng, [300, 300, 300], 19, 16, 1, 128)
    q = rng.standard_normal((3, 4, 128)).astype(np.float16)
    k0, v0 = cache.rows[0]
    k0[250] = 40 * q[0, 0] / np.linalg.norm(q[0, 0].astype(np.float64))
    k1, v1 = cache.rows[1]
    k1[:] = k1[0]
    k2, v2 = cache.rows[2]
    v2[123, 0, 5], v2[17, 0, 6], v2[290, 0, 7] = np.inf, -np.inf, np.nan
    for i, (k, v) in enumerate(cache.rows):
        for p in range(300):
            cache.key[cache.table[i, p // 16], p % 16] = k[p].view(np.uint16)
            cache.value[cache.table[i, p // 16], p % 16] = v[p].view(np.uint16)
    cache.owners = []
    cache.key_pages, cache.value_pages = cache.upload(cache.key), cache.upload(cache.value)
    cache.device_table = cache.upload_table()
    got = decode(ctx, cache, q, 4)
    clean = [(k0, v0), (k1, v1), (k2, np.where(np.isfinite(v2), v2, np.float16(0)))]
    cache.rows = clean
    want, tol = decode_want(cache, q)
    want[2, :, 5], want[2, :, 6], want[2, :, 7] = np.inf, -np.inf, np.nan
    g = f16(got).astype(np.float64)
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert (g[2, :, 5] == np.inf).all() and (g[2, :, 6] == -np.inf).all()
    finite = np.isfinite(want)
    assert (np.abs(g - want)[finite] <= tol[finite]).all()


# ------------------------------------------------------------- packed, paged --

def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.uint32)


def packed_want(q, k, v, starts, causal):
    outs = np.zeros(q.shape), np.zeros(q.shape)
    for a, e in zip(starts[:-1], starts[1:]):
        n = int(e) - int(a)
        seen = [np.arange(i + 1 if causal else n) for i in range(n)]
        for dst, src in zip(outs, attend(q[a:e].astype(np.float64), k[a:e], v[a:e], seen, True)):
            dst[a:e] = src
    return outs


COUNTS = [1, 0, 2, 33, 0, 64, 65, 7, 130, 1]


@pytest.mark.parametrize("hq,hkv,d,causal", [(8, 2, 128, True), (8, 2, 128, False), (5, 1, 64, True), (4, 4, 32, True),
                                             (3, 1, 256, True), (12, 4, 256, False), (40, 8, 128, True),
                                             (6, 2, 64, False), (16, 1, 32, True), (40, 1, 128, True)])
def test_packed_prompts(ctx, hq, hkv, d, causal):
    rng = np.random.default_rng(hq + d)
    starts = starts_of(COUNTS)
    n = int(starts[-1]) + 3  # three rows behind the last sequence
    qkv = rng.standard_normal((n, hq + 2 * hkv, d)).astype(np.float16)
    qkv[n - 3:] = poison(rng, (3, hq + 2 * hkv, d)).view(np.float16)
    owner, rows = padded_rows(ctx, qkv)
    stride = rows.strides[0]
    part = [rows.view((n, h, d), (stride, d, 1), offset=o * d) for h, o in ((hq, 0), (hkv, hq), (hkv, hq + hkv))]
    out = ctx.tensor(np.full((n, hq, d), 0x1234, np.uint16))
    batch = ctx.begin_batch()
    batch.attention_packed(*part, ctx.tensor(starts, U32), AttentionConfig(hq, hkv, d, causal, 9), out=out)
    batch.finish()
    got = ctx.download(out)
    assert (got[n - 3:] == 0x1234).all(), "rows behind the last sequence were written"
    e = n - 3
    hold(got[:e], *packed_want(qkv[:e, :hq], qkv[:e, hq:hq + hkv], qkv[:e, hq + hkv:], starts, causal))


def test_packed_longer_prompts_and_equal_calls(ctx):
    rng = np.random.default_rng(3)
    hq, hkv, d = 4, 2, 128
    starts = starts_of([700, 3, 500])
    n = int(starts[-1])
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    t = [ctx.tensor(x.view(np.uint16)) for x in (q, k, v)]
    s = ctx.tensor(starts, U32)
    got = []
    for _ in range(2):
        batch = ctx.begin_batch()
        out = batch.attention_packed(*t, s, AttentionConfig(hq, hkv, d))
        batch.finish()
        got.append(ctx.download(out))
    hold(got[0], *packed_want(q, k, v, starts, True))
    assert np.array_equal(got[0], got[1])


def test_packed_values_that_earlier_rows_must_not_see(ctx):
    """Infinities and NaN in a row's K and V reach that row and the later ones only."""
    rng = np.random.default_rng(4)
    for d, bad in ((128, 70), (64, 5), (32, 100), (256, 33)):
        n, hq, hkv = 140, 4, 1
        q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
        v[bad, 0, 3], v[bad + 1, 0, 4], v[bad + 2, 0, 5] = np.inf, -np.inf, np.nan
        k[bad + 30, 0, :] = np.nan
        starts = starts_of([n])
        batch = ctx.begin_batch()
        out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32),
                                     AttentionConfig(hq, hkv, d))
        batch.finish()
        got = ctx.download(out)
        clean = np.where(np.isfinite(v), v, np.float16(0))
        want, tol = packed_want(q, np.where(np.isnan(k), np.float16(0), k), clean, starts, True)
        hold(got[:bad], want[:bad], tol[:bad], f"d {d}: rows before")
        g = f16(got)
        near = slice(bad + 2, bad + 16)  # their weights are above f16's smallest value
        assert (g[near, :, 3] == np.inf).all() and (g[near, :, 4] == -np.inf).all() and np.isnan(g[near, :, 5]).all()
        rest = [c for c in range(d) if c not in (3, 4, 5)]
        hold(got[near][..., rest], want[near][..., rest], tol[near][..., rest], f"d {d}: other columns")
        assert np.isnan(g[bad + 30:]).all()


def paged_want(cache, q, starts, causal):
    want, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for i, (a, e) in enumerate(zip(starts[:-1], starts[1:])):
        n, total = int(e) - int(a), len(cache.rows[i][0])
        there = cache.there(i, total)
        seen = []
        for t in range(n):
            last = total - n + t if causal else total - 1
            seen.append(there[there <= last])
        want[a:e], tol[a:e] = attend(q[a:e].astype(np.float64), *cache.rows[i], seen, True)
    return want, tol


def paged(ctx, cache, q, starts, hq, causal=True):
    owner, view = padded_rows(ctx, q)
    out = ctx.tensor(np.full(q.shape, 0x1234, np.uint16))
    batch = ctx.begin_batch()
    batch.attention_paged(view, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                          ctx.tensor(starts, U32), AttentionConfig(hq, cache.hkv, cache.d, causal, 3), out=out)
    batch.finish()
    return ctx.download(out)


@pytest.mark.parametrize("hq,hkv,d,size,layout,causal", [
    (8, 2, 128, 16, "head_major", True), (8, 2, 128, 64, "gaps", False), (5, 1, 64, 32, "position_major", True),
    (4, 4, 32, 16, "gaps", True), (3, 1, 256, 16, "head_major", True), (40, 8, 128, 256, "position_major", True),
    (6, 2, 256, 128, "gaps", False), (24, 1, 64, 16, "head_major", True)])
def test_paged_rows_on_cached_keys(ctx, hq, hkv, d, size, layout, causal):
    rng = np.random.default_rng(hq + size)
    counts = [1, 0, 5, 32, 1, 70, 3, 16]
    cached = [0, 9, 63, 200, 330, 0, 64, 1]
    lengths = [a + b for a, b in zip(counts, cached)]
    cache = Cache(ctx, rng, lengths, -(-340 // size), size, hkv, d, layout)
    starts = starts_of(counts)
    q = (1.5 * rng.standard_normal((int(starts[-1]) + 2, hq, d))).astype(np.float16)
    got = paged(ctx, cache, q, starts, hq, causal)
    assert (got[-2:] == 0x1234).all()
    hold(got[:-2], *paged_want(cache, q[:-2], starts, causal))


def test_paged_long_cache(ctx):
    rng = np.random.default_rng(11)
    cache = Cache(ctx, rng, [3000, 1203, 2500], 200, 16, 2, 128)
    starts = starts_of([2, 130, 40])
    q = rng.standard_normal((172, 4, 128)).astype(np.float16)
    got = paged(ctx, cache, q, starts, 4)
    hold(got, *paged_want(cache, q, starts, True))
    assert np.array_equal(got, paged(ctx, cache, q, starts, 4))


@pytest.mark.parametrize("size", [16, 64])
def test_paged_without_some_pages(ctx, size):
    rng = np.random.default_rng(12)
    missing = [(0, 0), (0, 3), (1, 1), (2, 0), (2, 1), (2, 2), (2, 3)]
    cache = Cache(ctx, rng, [4 * size + 5, 3 * size, 4 * size, 20], 1600 // size, size, 1, 128, missing=missing)
    starts = starts_of([20, 17, 33, 20])
    q = rng.standard_normal((90, 2, 128)).astype(np.float16)
    want, tol = paged_want(cache, q, starts, True)
    assert np.isnan(want[37:70]).all()
    hold(paged(ctx, cache, q, starts, 2), want, tol)


def test_paged_more_rows_than_keys(ctx):
    """The first rows of such a sequence have no position: NaN. A sequence of length 0: all."""
    rng = np.random.default_rng(13)
    cache = Cache(ctx, rng, [3, 0, 40], 4, 16, 1, 64)
    starts = starts_of([5, 4, 2])
    q = rng.standard_normal((11, 2, 64)).astype(np.float16)
    want, tol = paged_want(cache, q, starts, True)
    assert np.isnan(want[:2]).all() and not np.isnan(want[2:5]).any() and np.isnan(want[5:9]).all()
    hold(paged(ctx, cache, q, starts, 2), want, tol)


def test_row_starts_out_of_order_stay_in_bounds(ctx):
    """Offsets past the rows are cut, and a sequence that ends before it starts is empty."""
    rng = np.random.default_rng(14)
    cache = Cache(ctx, rng, [20, 20, 20, 20], 4, 16, 1, 64)
    q = rng.standard_normal((10, 2, 64)).astype(np.float16)
    starts = np.array([2, 6, 4, 9, NOWHERE], np.uint32)  # rows 2-5, none, 4-8, 9
    got = paged(ctx, cache, q, starts, 2)
    assert (got[:2] == 0x1234).all()
    one = paged_want(cache, q, np.array([2, 6, 6, 6, 6]), True)
    hold(got[2:4], one[0][2:4], one[1][2:4])
    last = paged_want(cache, q, np.array([9, 9, 9, 9, 10]), True)
    hold(got[9:], last[0][9:], last[1][9:])


# ------------------------------------------------------------------- append --

def rotated(x, weight, position):
    """[n, H, D] in 64 bits at positions [n], and how far a kernel's f32 steps may be off: a
    few roundings of each product (the norm's sum of D squares: D 2^-24), the angle's
    fraction of a turn (2^-24 of a turn: 4e-7 of the pair's size) and its sine (2^-22)."""
    d = x.shape[-1]
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * weight.astype(np.float64)
    angle = position[:, None, None] * THETA ** (-2.0 * np.arange(d // 2) / d)
    a, b = x[..., :d // 2], x[..., d // 2:]
    r = np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)
    pair = np.hypot(a, b)
    off = np.concatenate([pair, pair], -1) * ((d + 8) * 2.0 ** -24 + 2.0 ** -20)
    return r, off + HALF_STEP * (np.abs(r) + off) + 2.0 ** -25


def append(ctx, cache, x, starts, weights, q_out=None):
    q, k, v = x
    n, hq, d = q.shape
    out = ctx.tensor(np.full(q.shape, 0x1234, np.uint16)) if q_out is None else q_out
    t = [padded_rows(ctx, a) for a in x]
    w = [ctx.tensor(a.view(np.uint16)) for a in weights] if weights is not None else [None, None]
    batch = ctx.begin_batch()
    batch.qk_norm_rope_paged(t[0][1], t[1][1], t[2][1], *w, cache.key_pages, cache.value_pages, cache.device_table,
                             cache.device_lengths, QkNormRopeCacheConfig(55, THETA, EPS),
                             row_starts=None if starts is None else ctx.tensor(starts, U32), out=out)
    batch.finish()
    return ctx.download(out)


def check_append(ctx, cache, x, starts, weights):
    q, k, v = x
    got = append(ctx, cache, x, starts, weights)
    key, value = cache.download(0), cache.download(1)
    want_key, want_value = cache.key.copy(), cache.value.copy()
    if starts is None:
        starts = np.arange(len(q) + 1)
    size, row_of = cache.size, {}
    for i, (a, e) in enumerate(zip(starts[:-1], starts[1:])):
        for r in range(a, e):
            position = int(cache.lengths[i]) - (int(e) - r)
            if position >= 0:
                row_of[r] = (cache.table[i, position // size], position % size, position)
    rows = np.array(sorted(row_of))
    at = np.array([row_of[r] for r in rows], np.int64)
    qw, kw = weights if weights is not None else (None, None)
    hold(got[rows], *rotated(q[rows], qw, at[:, 2]), "query")
    rest = np.setdiff1d(np.arange(len(q)), rows)
    assert (got[rest] == 0x1234).all(), "a row without a position was written"
    stored = at[:, 0] < cache.pages
    for r, (page, slot, _) in zip(rows[stored], at[stored]):
        want_value[page, slot] = v[r].view(np.uint16)
    assert np.array_equal(value, want_value), "value pages"
    want, tol = rotated(k[rows[stored]], kw, at[stored, 2])
    hold(key[at[stored, 0], at[stored, 1]], want, tol, "key")
    want_key[at[stored, 0], at[stored, 1]] = key[at[stored, 0], at[stored, 1]]
    assert np.array_equal(key, want_key), "another key slot was written"


def rows_for(rng, n, hq, hkv, d):
    x = tuple(rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    return x, tuple(rng.uniform(0.5, 2.0, d).astype(np.float16) for _ in "qk")


@pytest.mark.parametrize("hq,hkv,d,size,layout,norm", [
    (8, 2, 128, 16, "head_major", True), (5, 1, 64, 32, "gaps", True), (7, 7, 32, 16, "position_major", False),
    (3, 1, 256, 64, "gaps", True), (40, 8, 128, 16, "position_major", False), (16, 8, 128, 256, "head_major", True),
    (12, 4, 256, 16, "head_major", False), (64, 8, 64, 16, "gaps", True)])
@pytest.mark.parametrize("counts", [[1, 0, 2, 33, 0, 20, 1], [1] * 70])
def test_append_packed_rows(ctx, hq, hkv, d, size, layout, norm, counts):
    rng = np.random.default_rng(hq + d + size)
    cached = rng.integers(0, 150, len(counts))
    cache = Cache(ctx, rng, [int(a + b) for a, b in zip(counts, cached)], -(-200 // size), size, hkv, d, layout)
    starts = starts_of(counts)
    x, weights = rows_for(rng, int(starts[-1]) + 2, hq, hkv, d)
    check_append(ctx, cache, x, starts, weights if norm else None)


def test_append_one_row_per_sequence_and_lengths_of_zero(ctx):
    rng = np.random.default_rng(21)
    lengths = [1, 0, 17, 16, 64, 0, 33]
    cache = Cache(ctx, rng, lengths, 4, 16, 2, 128)
    x, weights = rows_for(rng, len(lengths), 8, 2, 128)
    check_append(ctx, cache, x, None, weights)


def test_append_far_positions(ctx):
    """Angles of 10^6 radians: 32-bit ones would be off by 0.06."""
    rng = np.random.default_rng(22)
    n, size, width = 4, 65536, 17
    lengths = [1_000_003, 131_072, 65_536, 999]
    table = np.full((n, width), NOWHERE, np.uint32)
    x, weights = rows_for(rng, n, 2, 1, 64)
    cache = Cache(ctx, rng, [1], 1, 16, 1, 64)  # storage of its own; the positions have no page
    cache.lengths, cache.table, cache.size = np.array(lengths), table, size
    pool = ctx.empty((1, size, 1, 64))
    cache.key_pages = cache.value_pages = pool
    owner = ctx.tensor(table, U32)
    cache.device_table, cache.device_lengths = owner, ctx.tensor(np.array(lengths, np.uint32), U32)
    got = append(ctx, cache, x, None, weights)
    hold(got, *rotated(x[0], weights[0], np.array(lengths) - 1))


def test_append_without_a_page_and_rows_without_a_position(ctx):
    rng = np.random.default_rng(23)
    cache = Cache(ctx, rng, [20, 3, 40], 4, 16, 2, 64, missing=[(0, 1), (2, 0), (2, 2)])
    starts = starts_of([10, 5, 40])
    x, weights = rows_for(rng, 55, 4, 2, 64)
    check_append(ctx, cache, x, starts, weights)


def test_append_in_place(ctx):
    rng = np.random.default_rng(24)
    cache = Cache(ctx, rng, [40, 12], 4, 16, 2, 128)
    starts = starts_of([30, 10])
    x, weights = rows_for(rng, 40, 4, 2, 128)
    want = append(ctx, cache, x, starts, weights)
    q = ctx.tensor(x[0].view(np.uint16))
    t = [ctx.tensor(a.view(np.uint16)) for a in (*x[1:], *weights)]
    batch = ctx.begin_batch()
    batch.qk_norm_rope_paged(q, *t, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                             QkNormRopeCacheConfig(0, THETA, EPS), row_starts=ctx.tensor(starts, U32), out=q)
    batch.finish()
    assert np.array_equal(ctx.download(q), want)


# ------------------------------------------------------------------ together --

@pytest.mark.parametrize("hq,hkv,d,size", [(8, 2, 128, 16), (4, 4, 64, 32), (4, 1, 256, 16), (6, 3, 32, 64)])
def test_a_server_of_three_sequences(ctx, hq, hkv, d, size):
    """Prompts (packed, and again through the pages), then a chunk, then single tokens, as one
    captured step replayed with new contents; one sequence of the batch stays empty."""
    rng = np.random.default_rng(31)
    counts, width = [37, 0, 90, 5], -(-160 // size)
    b = len(counts)
    cache = Cache(ctx, rng, [0] * b, width, size, hkv, d)
    order = rng.permutation(cache.pages)[:b * width].reshape(b, width).astype(np.uint32)
    cache.table = order
    cache.device_table = cache.upload_table()
    cfg, rope = AttentionConfig(hq, hkv, d), QkNormRopeCacheConfig(0, THETA, EPS)
    weights = tuple(rng.uniform(0.5, 2.0, d).astype(np.float16) for _ in "qk")
    w = [ctx.tensor(a.view(np.uint16)) for a in weights]
    held = [(np.zeros((0, hkv, d), np.float16), np.zeros((0, hkv, d), np.float16)) for _ in counts]

    def new_rows(counts):
        x = tuple(rng.standard_normal((sum(counts), h, d)).astype(np.float16) for h in (hq, hkv, hkv))
        for i, n in enumerate(counts):
            a = sum(counts[:i])
            position = len(held[i][0]) + np.arange(n)
            k = rotated(x[1][a:a + n], weights[1], position)[0].astype(np.float16)
            held[i] = (np.concatenate([held[i][0], k]), np.concatenate([held[i][1], x[2][a:a + n]]))
        return x

    def check(got, q_rot, counts, starts, f16_weights):
        """Against the held keys; a stored key may be one f16 step from the held one (its
        tolerance), which moves a score by 2^-10 sum |q k| at most."""
        for i, n in enumerate(counts):
            a, e = int(starts[i]), int(starts[i + 1])
            k, v = held[i]
            total = len(k)
            seen = [np.arange(total - n + t + 1) for t in range(n)]
            want, tol = attend(q_rot[a:e], k, v, seen, f16_weights)
            for t in range(n):
                for h in range(hq):
                    kk = k[seen[t], h // (hq // hkv)].astype(np.float64)
                    s = kk @ q_rot[a + t, h] / np.sqrt(d)
                    p = np.exp(s - s.max())
                    moved = 2.0 ** -10 * (np.abs(kk) @ np.abs(q_rot[a + t, h])).max() / np.sqrt(d)
                    tol[t, h] += 2 * moved * (p / p.sum()) @ np.abs(v[seen[t], h // (hq // hkv)].astype(np.float64))
            hold(got[a:e], want, tol, f"sequence {i}")

    # The prompts.
    x = new_rows(counts)
    starts, lengths = starts_of(counts), np.array([len(k) for k, _ in held], np.uint32)
    t = [ctx.tensor(a.view(np.uint16)) for a in x]
    dev_starts = ctx.tensor(starts, U32)
    ctx.upload(cache.device_lengths, lengths)
    batch = ctx.begin_batch()
    q = batch.qk_norm_rope_paged(*t, *w, cache.key_pages, cache.value_pages, cache.device_table,
                                 cache.device_lengths, rope, row_starts=dev_starts)
    through = batch.attention_paged(q, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                                    dev_starts, cfg)
    batch.finish()
    q_rot = f16(ctx.download(q)).astype(np.float64)
    check(ctx.download(through), q_rot, counts, starts, True)
    rotated_k = np.concatenate([k for k, _ in held])
    batch = ctx.begin_batch()
    direct = batch.attention_packed(q, ctx.tensor(rotated_k.view(np.uint16)), t[2], dev_starts, cfg)
    batch.finish()
    check(ctx.download(direct), q_rot, counts, starts, True)

    # A chunk, for two of the sequences.
    counts = [20, 0, 0, 40]
    x = new_rows(counts)
    starts, lengths = starts_of(counts), np.array([len(k) for k, _ in held], np.uint32)
    t = [ctx.tensor(a.view(np.uint16)) for a in x]
    dev_starts = ctx.tensor(starts, U32)
    ctx.upload(cache.device_lengths, lengths)
    batch = ctx.begin_batch()
    q = batch.qk_norm_rope_paged(*t, *w, cache.key_pages, cache.value_pages, cache.device_table,
                                 cache.device_lengths, rope, row_starts=dev_starts)
    out = batch.attention_paged(q, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                                dev_starts, cfg)
    batch.finish()
    check(ctx.download(out), f16(ctx.download(q)).astype(np.float64), counts, starts, True)

    # Single tokens: one captured step, replayed as the sequences grow (one has length 0).
    t = [ctx.empty((b, h, d)) for h in (hq, hkv, hkv)]
    q, out = ctx.empty((b, hq, d)), ctx.empty((b, hq, d))
    batch = ctx.begin_capture()
    batch.qk_norm_rope_paged(*t, *w, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                             rope, out=q)
    batch.attention_decode_paged(q, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                                 cfg, out=out)
    graph = batch.end_capture()
    for _ in range(4):
        counts = [1, 0, 1, 1]
        x = new_rows(counts)
        rows = [0, 2, 3]
        for dev, a in zip(t, x):
            full = poison(rng, (b,) + a.shape[1:])
            full[rows] = a.view(np.uint16)
            ctx.upload(dev, full)
        ctx.upload(cache.device_lengths, np.array([len(k) for k, _ in held], np.uint32))
        graph.launch()
        ctx.synchronize()
        got = ctx.download(out)
        assert np.isnan(f16(got[1])).all()
        check(got[rows], f16(ctx.download(q))[rows].astype(np.float64), counts, starts_of(counts), False)
    graph.destroy()


@pytest.mark.parametrize("kind", ["decode", "paged", "packed"])
def test_two_graphs_replayed_in_turn_match_eager_calls(ctx, kind):
    """Both take their workspaces from arenas of their own; replays alternate with eager calls."""
    rng = np.random.default_rng(41)
    hq, hkv, d = 8, 2, 128
    states = []
    for lengths, counts in (([900, 20, 333], [60, 20, 3]), ([5, 1200, 64, 700], [5, 2, 64, 90])):
        cache = Cache(ctx, rng, lengths, 80, 16, hkv, d)
        starts = starts_of([1] * len(lengths) if kind == "decode" else counts)
        q, k, v = (ctx.tensor(rng.standard_normal((int(starts[-1]), h, d)).astype(np.float16).view(np.uint16))
                   for h in (hq, hkv, hkv))
        states.append((cache, q, k, v, ctx.tensor(starts, U32), ctx.empty(q.shape)))
    cfg = AttentionConfig(hq, hkv, d)

    def enqueue(batch, state, out):
        cache, q, k, v, starts, _ = state
        pages = (cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths)
        if kind == "decode":
            batch.attention_decode_paged(q, *pages, cfg, out=out)
        elif kind == "paged":
            batch.attention_paged(q, *pages, starts, cfg, out=out)
        else:
            batch.attention_packed(q, k, v, starts, cfg, out=out)

    eager = []
    for state in states:
        batch = ctx.begin_batch()
        out = batch.empty(state[1].shape)
        enqueue(batch, state, out)
        batch.finish()
        eager.append(ctx.download(out))
    graphs = []
    for state in states:
        batch = ctx.begin_capture()
        enqueue(batch, state, state[-1])
        graphs.append(batch.end_capture())
    for _ in range(3):
        for state, graph in zip(states, graphs):
            ctx.upload(state[-1], np.zeros(state[-1].shape, np.uint16))
            graph.launch()
        batch = ctx.begin_batch()
        enqueue(batch, states[0], batch.empty(states[0][1].shape))
        batch.finish()
        for state, want in zip(states, eager):
            assert np.array_equal(ctx.download(state[-1]), want)
    for graph in graphs:
        graph.destroy()


def test_nothing_to_do(ctx):
    """No rows, or no sequences: nothing is launched and nothing written."""
    rng = np.random.default_rng(51)
    cache = Cache(ctx, rng, [5], 1, 16, 1, 64)
    cfg = AttentionConfig(2, 1, 64)
    q = ctx.tensor(np.full((3, 2, 64), 0x1234, np.uint16))
    kv = ctx.tensor(np.zeros((3, 1, 64), np.uint16))
    out = ctx.tensor(np.full((3, 2, 64), 0x4321, np.uint16))
    none = ctx.tensor(np.zeros(1, np.uint32), U32)
    empty = q.view((0, 2, 64), (128, 64, 1))
    ctx.set_kernel_profiling(True)
    try:
        batch = ctx.begin_batch()
        batch.attention_packed(q, kv, kv, none, cfg, out=out)
        batch.attention_packed(empty, kv.view((0, 1, 64), (64, 64, 1)), kv.view((0, 1, 64), (64, 64, 1)),
                               ctx.tensor(np.zeros(3, np.uint32), U32), cfg, out=empty)
        batch.finish()
        assert ctx.take_kernel_profiles() == []
    finally:
        ctx.set_kernel_profiling(False)
    assert (ctx.download(out) == 0x4321).all()


# ------------------------------------------------------- how the work is shared --

@pytest.mark.parametrize("hq,hkv,d,size,batch", [(16, 8, 128, 16, 20), (8, 8, 64, 32, 24), (4, 4, 32, 16, 40),
                                                 (8, 4, 256, 64, 33)])
def test_decode_of_many_units(ctx, hq, hkv, d, size, batch):
    """Enough (sequence, KV head) units that each wave walks a share of all tiles: shares that
    end inside a unit, units of one tile, of none, and one that many waves share."""
    rng = np.random.default_rng(61)
    lengths = [int(n) for n in rng.integers(0, 400, batch)]
    lengths[3], lengths[4], lengths[5], lengths[-1] = 2900, 0, 1, 0
    missing = [(3, p) for p in range(5, 2900 // size, 3)]
    cache = Cache(ctx, rng, lengths, -(-2900 // size), size, hkv, d, missing=missing)
    q = (1.5 * rng.standard_normal((batch, hq, d))).astype(np.float16)
    got = decode(ctx, cache, q, hq)
    hold(got, *decode_want(cache, q), f"decode {batch} x {hkv}")
    assert np.array_equal(got, decode(ctx, cache, q, hq)), "two calls differ"


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv,d", [(2, 1, 128), (4, 4, 64), (3, 1, 256)])
def test_packed_one_long_prompt_among_many(ctx, hq, hkv, d, causal):
    """More sequences than lanes, most of them empty or short, and two whose row tiles are cut."""
    rng = np.random.default_rng(62)
    counts = [int(n) for n in rng.integers(0, 4, 150)]
    counts[70], counts[149] = 1100, 600
    starts = starts_of(counts)
    n = int(starts[-1])
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    batch = ctx.begin_batch()
    out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32),
                                 AttentionConfig(hq, hkv, d, causal))
    batch.finish()
    hold(ctx.download(out), *packed_want(q, k, v, starts, causal))


@pytest.mark.parametrize("d,size", [(128, 16), (64, 32), (32, 16), (256, 16)])
@pytest.mark.parametrize("keys", [1100, 2500, 6000, 20000])
def test_paged_few_rows_on_a_long_cache(ctx, keys, d, size):
    """One row tile in up to 32 pieces, joined at once or in two steps, some of which see no
    key; the same when captured and replayed."""
    rng = np.random.default_rng(keys + d)
    pages = -(-keys // size)
    missing = [(0, p) for p in range(pages // 3, pages // 2)]
    cache = Cache(ctx, rng, [keys, 7], pages, size, 1, d, missing=missing)
    starts = starts_of([9, 2])
    q = rng.standard_normal((11, 5, d)).astype(np.float16)
    got = paged(ctx, cache, q, starts, 5)
    hold(got, *paged_want(cache, q, starts, True))
    t, s, out = ctx.tensor(q.view(np.uint16)), ctx.tensor(starts, U32), ctx.empty(q.shape)
    batch = ctx.begin_capture()
    batch.attention_paged(t, cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths, s,
                          AttentionConfig(5, 1, d), out=out)
    graph = batch.end_capture()
    for _ in range(3):
        ctx.upload(out, np.zeros(q.shape, np.uint16))
        graph.launch()
        ctx.synchronize()
        assert np.array_equal(ctx.download(out), got)
        assert np.array_equal(paged(ctx, cache, q, starts, 5), got)
    graph.destroy()


def test_more_sequences_than_one_launch_takes(ctx):
    rng = np.random.default_rng(63)
    hq, hkv, d, b = 2, 1, 64, 1100
    counts = [int(n) for n in rng.integers(0, 3, b)]
    counts[1030] = 70
    cached = rng.integers(0, 30, b)
    lengths = [int(a + c) for a, c in zip(counts, cached)]
    cache = Cache(ctx, rng, lengths, 7, 16, hkv, d)
    starts = starts_of(counts)
    n = int(starts[-1])
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    hold(paged(ctx, cache, q, starts, hq), *paged_want(cache, q, starts, True), "paged")
    batch = ctx.begin_batch()
    out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32),
                                 AttentionConfig(hq, hkv, d))
    batch.finish()
    hold(ctx.download(out), *packed_want(q, k, v, starts, True), "packed")
    q = rng.standard_normal((b, hq, d)).astype(np.float16)
    hold(decode(ctx, cache, q, hq), *decode_want(cache, q), "decode")
    x, weights = rows_for(rng, n, hq, hkv, d)
    check_append(ctx, cache, x, starts, weights)


def test_pages_past_four_gib(ctx):
    """Pools of 9 GB: the first page, the last, and one on either side of 2^32 bytes and of
    2^32 elements."""
    rng = np.random.default_rng(64)
    hq, hkv, d, size = 16, 8, 128, 64
    page = size * hkv * d
    pages = 2 ** 32 // page + 4000
    ids = [0, pages - 1, 2 ** 31 // page - 1, 2 ** 31 // page, 2 ** 32 // page - 1, 2 ** 32 // page]
    lengths, table = [160, 6 * size - 3], np.array([[1, 3, 5, 0, 0, 0], range(6)])
    store = [ctx.empty((pages, hkv, size, d)) for _ in "kv"]
    rows = []
    for t in store:
        kv = rng.standard_normal((6, size, hkv, d)).astype(np.float16)
        for at, one in zip(ids, kv):
            ctx.upload(t.view((hkv, size, d), (size * d, d, 1), offset=at * page),
                       np.ascontiguousarray(one.transpose(1, 0, 2)).view(np.uint16))
        rows.append(kv)
    views = [t.view((pages, size, hkv, d), (page, d, size * d, 1)) for t in store]
    held = [tuple(kv[table[i]].reshape(-1, hkv, d)[:n] for kv in rows) for i, n in enumerate(lengths)]
    dev_table = ctx.tensor(np.array(ids, np.uint32)[table], U32)
    dev_lengths = ctx.tensor(np.array(lengths, np.uint32), U32)
    cfg = AttentionConfig(hq, hkv, d)
    counts = [20, 3]
    starts = starts_of(counts)
    q = rng.standard_normal((23, hq, d)).astype(np.float16)
    new = [rng.standard_normal((2, h, d)).astype(np.float16) for h in (hq, hkv, hkv)]
    one, many = ctx.tensor(q[:2].view(np.uint16)), ctx.tensor(q.view(np.uint16))
    batch = ctx.begin_batch()
    a = batch.attention_decode_paged(one, *views, dev_table, dev_lengths, cfg)
    c = batch.attention_paged(many, *views, dev_table, dev_lengths, ctx.tensor(starts, U32), cfg)
    batch.qk_norm_rope_paged(*[ctx.tensor(x.view(np.uint16)) for x in new], None, None, *views, dev_table, dev_lengths,
                             QkNormRopeCacheConfig(0, THETA, EPS))
    batch.finish()
    got_one, got_many = ctx.download(a), ctx.download(c)
    for i, (k, v) in enumerate(held):
        n = len(k)
        hold(got_one[i:i + 1], *attend(q[i:i + 1].astype(np.float64), k, v, [np.arange(n)], False), "decode")
        s, e = starts[i], starts[i + 1]
        seen = [np.arange(n - counts[i] + t + 1) for t in range(counts[i])]
        hold(got_many[s:e], *attend(q[s:e].astype(np.float64), k, v, seen, True), "paged")
        at, slot = ids[table[i][(n - 1) // size]], (n - 1) % size
        last = [ctx.download(t.view((hkv, d), (size * d, 1), offset=at * page + slot * d)) for t in store]
        assert np.array_equal(last[1], new[2][i].view(np.uint16)), "value"
        hold(last[0], *[x[0] for x in rotated(new[1][i:i + 1], None, np.array([n - 1]))], "key")


# ------------------------------------------------------------ layouts, sharing --

def spread_out(ctx, n, h, d):
    """An output in head-major storage with a gap between rows: (owner, view of [n, h, d])."""
    owner = ctx.tensor(np.full((h, n, d + 8), 0x1234, np.uint16))
    return owner, owner.view((n, h, d), (d + 8, n * (d + 8), 1))


@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 128), (5, 5, 64), (4, 1, 256), (8, 4, 32)])
def test_outputs_and_queries_in_other_layouts(ctx, hq, hkv, d):
    """Head-major queries and outputs with gaps, of which nothing but the rows is written; keys
    and values of one head that all KV heads share (a head stride of 0)."""
    rng = np.random.default_rng(71)
    counts, cached = [3, 1, 40], [20, 700, 0]
    starts = starts_of(counts)
    n = int(starts[-1])
    cache = Cache(ctx, rng, [a + b for a, b in zip(counts, cached)], 50, 16, hkv, d, "gaps")
    q = rng.standard_normal((n, hq, d)).astype(np.float16)
    store = np.full((hq, n, d + 16), 0x7E00, np.uint16)
    store[:, :, :d] = q.view(np.uint16).transpose(1, 0, 2)
    owner = ctx.tensor(store)
    view = owner.view((n, hq, d), (d + 16, n * (d + 16), 1))
    pages = (cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths)
    k, v = (rng.standard_normal((n, 1, d)).astype(np.float16) for _ in "kv")
    shared = [ctx.tensor(x.view(np.uint16)) for x in (k, v)]
    outs = [spread_out(ctx, n, hq, d), spread_out(ctx, n, hq, d), spread_out(ctx, 3, hq, d)]
    cfg, dev_starts = AttentionConfig(hq, hkv, d), ctx.tensor(starts, U32)
    batch = ctx.begin_batch()
    batch.attention_paged(view, *pages, dev_starts, cfg, out=outs[0][1])
    batch.attention_packed(view, *[t.view((n, hkv, d), (d, 0, 1)) for t in shared], dev_starts, cfg, out=outs[1][1])
    batch.attention_decode_paged(owner.view((3, hq, d), (d + 16, n * (d + 16), 1)), *pages, cfg, out=outs[2][1])
    batch.finish()
    wants = (paged_want(cache, q, starts, True),
             packed_want(q, np.repeat(k, hkv, 1), np.repeat(v, hkv, 1), starts, True), decode_want(cache, q[:3]))
    for (store, _), (want, tol) in zip(outs, wants):
        raw = ctx.download(store)
        assert (raw[:, :, d:] == 0x1234).all(), "the gap between rows was written"
        hold(raw[:, :, :d].transpose(1, 0, 2), want, tol)


def test_sequences_that_share_pages(ctx):
    """A prompt's pages in three tables, each with a page of its own behind them."""
    rng = np.random.default_rng(72)
    hq, hkv, d, size = 8, 2, 128, 16
    cache = Cache(ctx, rng, [100, 100, 100], 7, size, hkv, d)
    cache.table[1:, :6] = cache.table[0, :6]
    cache.device_table = cache.upload_table()
    for i in (1, 2):
        cache.rows[i] = tuple(np.concatenate([a[:96], b[96:]]) for a, b in zip(cache.rows[0], cache.rows[i]))
    q = rng.standard_normal((3, hq, d)).astype(np.float16)
    hold(decode(ctx, cache, q, hq), *decode_want(cache, q))
    starts = starts_of([4, 4, 4])
    q = rng.standard_normal((12, hq, d)).astype(np.float16)
    hold(paged(ctx, cache, q, starts, hq), *paged_want(cache, q, starts, True))


def test_two_contexts_at_once(ctx):
    """Calls of two contexts in flight together, each with pieces to join, match single ones."""
    rng = np.random.default_rng(73)
    hq, hkv, d = 8, 2, 128
    other = mi_attn.Context(0)
    try:
        sides = []
        for c in (ctx, other):
            cache = Cache(c, rng, [3000, 900, 40], 190, 16, hkv, d)
            starts = starts_of([1, 60, 3])
            q = rng.standard_normal((64, hq, d)).astype(np.float16)
            sides.append((c, cache, c.tensor(q.view(np.uint16)), c.tensor(starts, U32), q, starts))
        cfg = AttentionConfig(hq, hkv, d)

        def enqueue(side):
            c, cache, t, dev_starts, _, _ = side
            pages = (cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths)
            batch = c.begin_batch()
            out = [c.empty((64, hq, d)), c.empty((3, hq, d))]
            for _ in range(5):
                batch.attention_paged(t, *pages, dev_starts, cfg, out=out[0])
                batch.attention_decode_paged(t.view((3, hq, d), (hq * d, d, 1)), *pages, cfg, out=out[1])
            return batch, out

        alone = []
        for side in sides:
            batch, out = enqueue(side)
            batch.finish()
            alone.append([side[0].download(o) for o in out])
            hold(alone[-1][0], *paged_want(side[1], side[4], side[5], True))
        both = [enqueue(side) for side in sides]
        for batch, _ in both:
            batch.finish()
        for side, (_, out), want in zip(sides, both, alone):
            for o, w in zip(out, want):
                assert np.array_equal(side[0].download(o), w)
        del both, sides, out, o
    finally:
        other.close()


@pytest.mark.parametrize("hq,hkv,d,size,batch,low,high", [
    (16, 16, 64, 16, 70, 0, 128), (64, 32, 32, 16, 70, 100, 260), (16, 8, 128, 16, 300, 0, 33), (16, 16, 256, 16, 40, 1, 60)])
def test_decode_of_many_short_units(ctx, hq, hkv, d, size, batch, low, high):
    """More units than workgroups, each a wave's own; several in turn; some without a key."""
    rng = np.random.default_rng(65)
    lengths = [int(n) for n in rng.integers(low, high, batch)]
    cache = Cache(ctx, rng, lengths, -(-high // size), size, hkv, d, missing=[(1, 0), (batch - 1, 0)])
    q = (1.5 * rng.standard_normal((batch, hq, d))).astype(np.float16)
    got = decode(ctx, cache, q, hq)
    hold(got, *decode_want(cache, q), f"decode {batch} x {hkv}")
    assert np.array_equal(got, decode(ctx, cache, q, hq)), "two calls differ"


@pytest.mark.parametrize("hq,hkv", [(4096, 4096), (4200, 4200), (130, 1), (1030, 103)])
def test_many_heads(ctx, hq, hkv):
    """As many KV heads as a decode launch takes, more than the pieces' counters reach (packed
    rows only), and groups that are no multiple of a chunk; a sample of the heads is checked."""
    rng = np.random.default_rng(81)
    d, size, counts = 32, 16, [3, 0, 70]
    starts = starts_of(counts)
    n = int(starts[-1])
    heads = np.unique(np.concatenate([[0, hq - 1], rng.integers(0, hq, 6)]))
    kv = heads // (hq // hkv)
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    cfg = AttentionConfig(hq, hkv, d)
    batch = ctx.begin_batch()
    out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32), cfg)
    batch.finish()
    hold(ctx.download(out)[:, heads], *packed_want(q[:, heads], k[:, kv], v[:, kv], starts, True), "packed")
    if hkv > 4096:
        return
    cache = Cache(ctx, rng, [130, 0, 33], 9, size, hkv, d)
    q = rng.standard_normal((3, hq, d)).astype(np.float16)
    got = decode(ctx, cache, q, hq)[:, heads]
    cache.rows = [(k[:, kv], v[:, kv]) for k, v in cache.rows]
    hold(got, *decode_want(cache, q[:, heads]), "decode")


def test_one_graph_for_every_division_of_the_work(ctx):
    """Captured once, replayed on lengths and row offsets that the kernels divide in every way
    (none, short, equal, ragged, one long), each time as the eager call on them."""
    rng = np.random.default_rng(91)
    hq, hkv, d, size, b, n = 16, 8, 64, 16, 80, 300
    cache = Cache(ctx, rng, [1500] * b, 94, size, hkv, d)
    pages = (cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths)
    one = ctx.tensor(rng.standard_normal((b, hq, d)).astype(np.float16).view(np.uint16))
    q, k, v = (ctx.tensor(rng.standard_normal((n, h, d)).astype(np.float16).view(np.uint16)) for h in (hq, hkv, hkv))
    dev_starts = ctx.tensor(np.zeros(b + 1, np.uint32), U32)
    cfg = AttentionConfig(hq, hkv, d)

    def enqueue(batch, outs):
        batch.attention_decode_paged(one, *pages, cfg, out=outs[0])
        batch.attention_paged(q, *pages, dev_starts, cfg, out=outs[1])
        batch.attention_packed(q, k, v, dev_starts, cfg, out=outs[2])

    def outputs():
        return [ctx.tensor(np.full(t.shape, 0x1234, np.uint16)) for t in (one, q, q)]

    captured = outputs()
    batch = ctx.begin_capture()
    enqueue(batch, captured)
    graph = batch.end_capture()
    ragged = rng.integers(0, 1501, b)
    one_long = np.where(np.arange(b) == 7, 1500, 3)
    few = np.where(np.arange(b) < 4, 1500, 0)
    rows = {"none": np.zeros(b, int), "one": np.where(np.arange(b) == 7, n, 0), "each": np.full(b, 3),
            "some": np.where(np.arange(b) % 11 == 0, 30, 0)}
    for lengths, counts in ((np.zeros(b, int), "none"), (np.full(b, 20), "each"), (np.full(b, 1500), "each"),
                            (ragged, "some"), (one_long, "one"), (few, "one"), (np.full(b, 300), "some"),
                            (ragged, "each")):
        ctx.upload(cache.device_lengths, lengths.astype(np.uint32))
        ctx.upload(dev_starts, starts_of(rows[counts]))
        for t in captured:
            ctx.upload(t, np.full(t.shape, 0x1234, np.uint16))
        graph.launch()
        ctx.synchronize()
        eager = outputs()
        batch = ctx.begin_batch()
        enqueue(batch, eager)
        batch.finish()
        for t, e in zip(captured, eager):
            assert np.array_equal(ctx.download(t), ctx.download(e)), counts
        got = ctx.download(captured[0])
        for i in rng.integers(0, b, 3):
            key, value = cache.rows[i]
            want, tol = attend(f16(ctx.download(one))[i:i + 1].astype(np.float64), key, value,
                               [np.arange(int(lengths[i]))], False)
            hold(got[i:i + 1], want, tol)
    graph.destroy()
