"""NaN and infinities in keys and values that rows see, wherever the work is divided: a sum
with a NaN in it is NaN, and a positive weight, however small, leaves an infinity what it is."""
from __future__ import annotations

import numpy as np
import pytest

from mi_attn import U32, AttentionConfig
from helpers import f16
from test_gpu_paged import Cache, attend, decode, hold, paged, starts_of

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
