"""NaN and infinities in keys and values that rows see, wherever the work is divided: a sum
with a NaN in it is NaN, and a positive weight, however small, leaves an infinity what it is."""
from __future__ import annotations

import numpy as np
import pytest

from mi_attn import U32, AttentionConfig
from helpers import f16
from test_gpu_paged import Cache, attend, decode, hold, packed_want, paged, starts_of

pytestmark = pytest.mark.gpu


def stored(cache):
    """The cache on the device again, after its rows were changed on the host."""
    for i, (k, v) in enumerate(cache.rows):
        at = np.arange(len(k))
        pages = cache.table[i, at // cache.size]
        there = pages < cache.pages
        cache.key[pages[there], at[there] % cache.size] = k[there].view(np.uint16)
        cache.value[pages[there], at[there] % cache.size] = v[there].view(np.uint16)
    cache.owners = []
    cache.key_pages, cache.value_pages = cache.upload(cache.key), cache.upload(cache.value)
    cache.device_table = cache.upload_table()
    return cache


def packed(ctx, q, k, v, starts, causal=True):
    batch = ctx.begin_batch()
    out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32),
                                 AttentionConfig(q.shape[1], k.shape[1], q.shape[2], causal))
    batch.finish()
    return f16(ctx.download(out))


# ----------------------------------------------------------------- NaN in keys --

@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("lengths,hq,hkv", [
    ([129], 8, 8),                                    # pieces of four tiles and of one key
    ([33, 65, 97, 129, 161, 257, 1025], 8, 2),
    ([32 * n + 1 for n in range(1, 70)], 16, 8),      # shares that end where a tile of one key begins
    ([3001, 40] + [33] * 60, 16, 16)])
def test_decode_nan_in_the_newest_key(ctx, d, lengths, hq, hkv):
    """A piece of that key alone has no score but NaN, and makes the row NaN all the same."""
    rng = np.random.default_rng(d + len(lengths))
    cache = Cache(ctx, rng, lengths, -(-max(lengths) // 16), 16, hkv, d)
    spared = len(lengths) // 2 if len(lengths) > 1 else -1
    for i, (k, _) in enumerate(cache.rows):
        if i != spared:
            k[-1, :, 3] = np.nan
    stored(cache)
    q = rng.standard_normal((len(lengths), hq, d)).astype(np.float16)
    got = decode(ctx, cache, q, hq)
    for i in range(len(lengths)):
        if i != spared:
            assert np.isnan(f16(got[i])).all(), f"length {lengths[i]}"
        else:
            k, v = cache.rows[i]
            hold(got[i:i + 1], *attend(q[i:i + 1].astype(np.float64), k, v, [np.arange(len(k))], False))


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_decode_nan_in_every_key_of_some_tiles(ctx, d):
    rng = np.random.default_rng(d)
    lengths = [6000, 700, 90]
    cache = Cache(ctx, rng, lengths, 6000 // 16, 16, 2, d)
    cache.rows[0][0][1000:3000] = np.nan
    cache.rows[1][0][:128] = np.nan
    stored(cache)
    q = rng.standard_normal((3, 4, d)).astype(np.float16)
    got = f16(decode(ctx, cache, q, 4))
    assert np.isnan(got[:2]).all() and not np.isnan(got[2]).any()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("keys", [2500, 6000])
def test_paged_nan_in_every_key_of_the_last_pieces(ctx, d, keys):
    """NaN from a tile's first key to the end, for many tiles: wherever the last piece begins, and
    the last few that are joined first (6000 keys), one sequence has NaN there and nowhere else."""
    rng = np.random.default_rng(d + keys)
    b, tile = 14, 32 if d == 256 else 64
    cache = Cache(ctx, rng, [keys] * b, keys // 16 + 1, 16, 1, d)
    clean = cache.rows
    q = rng.standard_normal((b, 5, d)).astype(np.float16)
    for start in range(0, 42 if keys == 6000 else 14, b - 1):
        cache.rows = [(k.copy(), v) for k, v in clean]
        for i in range(1, b):
            cache.rows[i][0][(keys // tile - start - i + 1) * tile:] = np.nan
        stored(cache)
        got = f16(paged(ctx, cache, q, starts_of([1] * b), 5))
        assert np.isfinite(got[0]).all() and np.isnan(got[1:]).all(), f"from tile -{start}"


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_nan_in_every_key_of_the_last_pieces(ctx, d, causal):
    rng = np.random.default_rng(d)
    n = 1150
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (2, 1, 1))
    for first in range(n - n % 32, n - 420, -32):
        bad = k.copy()
        bad[first:] = np.nan
        got = packed(ctx, q, bad, v, starts_of([n]), causal)
        at = first if causal else 0
        assert np.isfinite(got[:at]).all() and np.isnan(got[at:]).all(), f"from key {first}"


# -------------------------------------------------- infinities of small weights --

def far(rng, n, hq, hkv, d, seen, gap):
    """q, k, v of n keys of which those of `seen` have scores `gap` below the others'."""
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))
    q[:, :, 0], k[:, :, 0] = 8, 0
    k[seen, :, 0] = -gap * np.sqrt(d) / 8
    return q, k, v


GAPS = [25.0, 60.0, 200.0]  # weights of 2^-36, 2^-87 and 2^-289 of the largest


def check_infinite(got, lim, at):
    """Rows got [n, H, D], which see keys up to lim[i]: columns 3 to 6."""
    for key, what, col in ((at[0], np.inf, 3), (at[1], -np.inf, 4)):
        sees = lim >= key
        assert (got[sees][..., col] == what).all() and np.isfinite(got[~sees][..., col]).all()
    sees = lim >= at[2]
    assert np.isnan(got[sees][..., 5]).all() and np.isfinite(got[~sees][..., 5]).all()
    both, one = lim >= max(at[0], at[1]), (lim >= min(at[0], at[1])) & (lim < max(at[0], at[1]))
    assert np.isnan(got[both][..., 6]).all() and np.isinf(got[one][..., 6]).all()
    rest = [c for c in range(got.shape[-1]) if not 3 <= c <= 6]
    assert np.isfinite(got[..., rest]).all()


def put_infinite(v, at):
    v[at[0], :, 3], v[at[1], :, 4], v[at[2], :, 5] = np.inf, -np.inf, np.nan
    v[at[0], :, 6], v[at[1], :, 6] = np.inf, -np.inf


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("d,n", [(32, 300), (64, 300), (128, 300), (256, 300), (128, 1300), (256, 1300)])
def test_packed_infinities_of_small_weights(ctx, d, n, gap):
    """In whole tiles, which need no mask, and in the pieces of cut row tiles (1300 rows)."""
    rng = np.random.default_rng(d)
    at = [70, 40, 100]
    q, k, v = far(rng, n, 4, 2, d, at, gap)
    put_infinite(v, at)
    got = packed(ctx, q, k, v, starts_of([n]))
    check_infinite(got, np.arange(n), at)
    got = packed(ctx, q, k, v, starts_of([n]), causal=False)
    check_infinite(got, np.full(n, n - 1), at)
    clean = np.where(np.isfinite(v), v, np.float16(0))
    want, tol = packed_want(q, k, clean, starts_of([n]), True)
    rest = [c for c in range(d) if not 3 <= c <= 6]
    got = packed(ctx, q, k, v, starts_of([n]))
    assert (np.abs(got - want)[..., rest] <= tol[..., rest]).all()


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("keys", [900, 6000])
def test_paged_infinities_of_small_weights(ctx, d, keys, gap):
    rng = np.random.default_rng(d + keys)
    at = [keys // 2, 130, keys - 20]
    q, k, v = far(rng, keys, 4, 1, d, at, gap)
    put_infinite(v, at)
    cache = Cache(ctx, rng, [keys, 50], keys // 16 + 1, 16, 1, d, missing=[(0, 20)])
    cache.rows[0] = (k, v)
    cache.rows[1][1][10:] = np.nan
    stored(cache)
    starts = starts_of([40, 45])
    q = np.concatenate([q[:40], rng.standard_normal((45, 4, d)).astype(np.float16)])
    got = f16(paged(ctx, cache, q, starts, 4))
    check_infinite(got[:40], keys - 40 + np.arange(40), at)
    assert np.isfinite(got[40:45]).all() and np.isnan(got[45:]).all()  # its rows see 6 to 50 keys


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("keys,batch,hkv", [(90, 1, 1), (4000, 1, 2), (333, 70, 16), (40, 70, 16)])
def test_decode_infinities_of_small_weights(ctx, d, keys, batch, hkv, gap):
    """One piece, pieces of workgroups, shares of waves and whole units."""
    rng = np.random.default_rng(d + keys)
    at = [keys // 2, 3, keys - 2]
    q, k, v = far(rng, keys, hkv, hkv, d, at, gap)
    put_infinite(v, at)
    lengths = [keys] * batch
    if batch > 60:
        lengths[5], lengths[9] = 3 * keys, 0
    cache = Cache(ctx, rng, lengths, -(-max(lengths) // 16), 16, hkv, d)
    for i in range(batch):
        if lengths[i] == keys:
            cache.rows[i] = (k, v)
    stored(cache)
    got = f16(decode(ctx, cache, np.repeat(q[:1], batch, 0), hkv))
    for i in range(batch):
        if lengths[i] == keys:
            check_infinite(got[i:i + 1], np.array([keys - 1]), at)
    if batch > 60:
        assert np.isfinite(got[5]).all() and np.isnan(got[9]).all()


# ---------------------------------------------------------- no finite score at all --

def without_scores(ctx, d, lengths, hkv=1):
    """A cache whose keys are -inf where the queries are 1, but for the last sequence's."""
    rng = np.random.default_rng(d)
    cache = Cache(ctx, rng, lengths, -(-max(lengths) // 16), 16, hkv, d)
    for k, _ in cache.rows[:-1]:
        k[:, :, 0] = -np.inf
    q = rng.standard_normal((len(lengths), 2 * hkv, d)).astype(np.float16)
    q[:, :, 0] = 1
    return stored(cache), q


@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("lengths,hkv", [([1, 40, 3000, 20], 1), ([1, 40, 0, 120] * 30 + [70], 8), ([900, 1, 40] * 20 + [70], 16)])
def test_decode_rows_whose_scores_are_all_minus_infinity(ctx, d, lengths, hkv):
    """The weights of such a row are 0 / 0."""
    cache, q = without_scores(ctx, d, lengths, hkv)
    got = f16(decode(ctx, cache, q, 2 * hkv))
    assert np.isnan(got[:-1]).all() and np.isfinite(got[-1]).all()


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_paged_rows_whose_scores_are_all_minus_infinity(ctx, d):
    cache, q = without_scores(ctx, d, [1, 40, 3000, 20])
    got = f16(paged(ctx, cache, q, starts_of([1, 1, 1, 1]), 2))
    assert np.isnan(got[:3]).all() and np.isfinite(got[3]).all()
