"""NaN and infinities in keys and values that rows see, wherever the work is divided: a sum
with a NaN in it is NaN, and a positive weight, however small, leaves an infinity what it is."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import f16
from test_gpu_paged import Cache, attend, decode, hold

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
