"""Sequences that are longer than their rows of the block table: a position past the table has no
page, as one whose table entry names none."""
from __future__ import annotations

import numpy as np
import pytest

from mi_attn import U32, AttentionConfig
from helpers import f16
from test_gpu_paged import (NOWHERE, Cache, append, attend, hold, paged, rotated, rows_for,
                            starts_of)

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


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv,d,size", [(4, 2, 128, 16), (5, 1, 64, 32), (3, 1, 256, 16), (4, 4, 32, 64)])
def test_paged_rows_past_the_table(ctx, hq, hkv, d, size, causal):
    """A row sees the keys up to its position that the table can name."""
    rng = np.random.default_rng(d + size)
    width = 1280 // size
    full = width * size
    cache = Cache(ctx, rng, [full, full, full, full, 40], width, size, hkv, d)
    lengths = np.array([full + 5, full + 1000, NOWHERE, full, 40], np.int64)
    counts = [70, 3, 40, 20, 60]  # of the last, 20 rows have no position
    ctx.upload(cache.device_lengths, lengths.astype(np.uint32))
    starts = starts_of(counts)
    q = rng.standard_normal((int(starts[-1]), hq, d)).astype(np.float16)
    got = paged(ctx, cache, q, starts, hq, causal)
    for i, n in enumerate(counts):
        a, e = starts[i], starts[i + 1]
        k, v = cache.rows[i]
        seen = [np.arange(max(0, min(len(k), lengths[i] - n + t + 1 if causal else lengths[i]))) for t in range(n)]
        hold(got[a:e], *attend(q[a:e].astype(np.float64), k, v, seen, True), f"sequence {i}")


def test_a_sequence_that_outgrows_its_table(ctx):
    """Appended and read token by token past the end: the stored keys stay, and are all seen."""
    rng = np.random.default_rng(2)
    hq, hkv, d, size = 4, 2, 128, 16
    cache = Cache(ctx, rng, [30], 2, size, hkv, d)
    held = [[r] for r in cache.rows[0]]
    cfg = AttentionConfig(hq, hkv, d)
    for length in range(31, 37):
        ctx.upload(cache.device_lengths, np.array([length], np.uint32))
        x, weights = rows_for(rng, 1, hq, hkv, d)
        q = append(ctx, cache, x, None, weights)
        if length <= 32:
            page = cache.table[0, (length - 1) // size], (length - 1) % size
            held[0].append(cache.download(0)[page][None].view(np.float16))
            held[1].append(x[2])
        k, v = (np.concatenate(h) for h in held)
        assert len(k) == min(length, 32)
        out = ctx.empty((1, hq, d))
        batch = ctx.begin_batch()
        batch.attention_paged(ctx.tensor(q), cache.key_pages, cache.value_pages, cache.device_table, cache.device_lengths,
                              ctx.tensor(starts_of([1]), U32), cfg, out=out)
        one = batch.attention_decode_paged(ctx.tensor(q), cache.key_pages, cache.value_pages, cache.device_table,
                                           cache.device_lengths, cfg)
        batch.finish()
        q64 = f16(q).astype(np.float64)
        hold(ctx.download(out), *attend(q64, k, v, [np.arange(len(k))], True))
        hold(ctx.download(one), *attend(q64, k, v, [np.arange(len(k))], False))
