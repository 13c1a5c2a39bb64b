"""Sequences that are longer than their rows of the block table: a position past the table has no
page, as one whose table entry names none."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_paged import Cache, append, hold, rotated, rows_for, starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,size,layout", [(8, 2, 128, 16, "head_major"), (4, 4, 64, 32, "position_major"),
                                                  (5, 1, 256, 16, "gaps"), (6, 2, 32, 64, "head_major")])
def test_append_past_the_table(ctx, hq, hkv, d, size, layout):
    """Rows past the table are rotated at their own position and stored nowhere; those before it
    land where they belong, and no slot that was filled before changes."""
    rng = np.random.default_rng(d + size)
    width = 3
    full = width * size
    cache = Cache(ctx, rng, [full, full, full, 10], width, size, hkv, d, layout)
    lengths = np.array([full + 1, full + 7, full + 100_000, 10], np.int64)
    counts = [1, 12, 20, 4]  # the second sequence's first five rows have pages
    ctx.upload(cache.device_lengths, lengths.astype(np.uint32))
    starts = starts_of(counts)
    x, weights = rows_for(rng, int(starts[-1]), hq, hkv, d)
    got = append(ctx, cache, x, starts, weights)
    position = np.concatenate([n - c + np.arange(c) for n, c in zip(lengths, counts)])
    sequence = np.repeat(np.arange(4), counts)
    hold(got, *rotated(x[0], weights[0], position), "query")
    key, value = cache.download(0), cache.download(1)
    want_key, want_value = cache.key.copy(), cache.value.copy()
    for r in np.flatnonzero(position < full):
        at = cache.table[sequence[r], position[r] // size], position[r] % size
        want_value[at] = x[2][r].view(np.uint16)
        hold(key[at][None], *rotated(x[1][r:r + 1], weights[1], position[r:r + 1]), "key")
        want_key[at] = key[at]
    assert np.array_equal(value, want_value) and np.array_equal(key, want_key), "another slot was written"


def test_append_one_row_past_the_table(ctx):
    rng = np.random.default_rng(1)
    cache = Cache(ctx, rng, [32, 32, 32], 2, 16, 2, 128)
    lengths = np.array([33, 32, 0x7FFFFFFF], np.int64)
    ctx.upload(cache.device_lengths, lengths.astype(np.uint32))
    x, weights = rows_for(rng, 3, 4, 2, 128)
    hold(append(ctx, cache, x, None, weights), *rotated(x[0], weights[0], lengths - 1), "query")
    want = cache.value.copy()
    want[cache.table[1, 1], 15] = x[2][1].view(np.uint16)
    assert np.array_equal(cache.download(1), want)
