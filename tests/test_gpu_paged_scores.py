"""Packed and paged attention where the scores' reference has to move late: a key far above the
rest in a whole tile, in a masked one and in a piece of a cut row tile, and scores that grow from
tile to tile."""
from __future__ import annotations

import numpy as np
import pytest

from mi_attn import U32, AttentionConfig
from test_gpu_paged import Cache, hold, packed_want, paged, paged_want, starts_of
from test_gpu_paged_not_finite import stored

pytestmark = pytest.mark.gpu
DIMS = [32, 64, 128, 256]


def toward(q, k, at, score):
    """Keys `at` of k [L, Hkv, D] with the scaled score `score` (one per key) for every row: q's
    first value is 8 and k's 0 everywhere else."""
    d = q.shape[-1]
    q[..., 0], k[..., 0] = 8, 0
    k[at, :, 0] = (np.asarray(score) * np.sqrt(d) / 8)[..., None] if np.ndim(score) else score * np.sqrt(d) / 8


def packed_case(ctx, q, k, v, starts, causal=True):
    batch = ctx.begin_batch()
    out = batch.attention_packed(*[ctx.tensor(x.view(np.uint16)) for x in (q, k, v)], ctx.tensor(starts, U32),
                                 AttentionConfig(q.shape[1], k.shape[1], q.shape[2], causal))
    batch.finish()
    hold(ctx.download(out), *packed_want(q, k, v, starts, causal))


def normal(rng, n, hq, hkv, d):
    return tuple(rng.standard_normal((n, h, d)).astype(np.float16) for h in (hq, hkv, hkv))


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("score", [20.0, 40.0, -40.0])
@pytest.mark.parametrize("at", [[200], [30, 110, 290], [0], [299]])
def test_packed_a_key_far_from_the_rest(ctx, d, score, at):
    """Seen by whole tiles (early keys of late rows) and by masked ones (the rows next to it)."""
    rng = np.random.default_rng(d)
    q, k, v = normal(rng, 300, 3, 1, d)
    toward(q, k, at, score)
    packed_case(ctx, q, k, v, starts_of([300]))
    packed_case(ctx, q, k, v, starts_of([300]), causal=False)


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("step", [0.2, 0.5, -0.5])
def test_packed_scores_that_grow(ctx, d, step):
    """Over 420 keys, 16 at a time: the reference moves several times, or never again."""
    rng = np.random.default_rng(d)
    q, k, v = normal(rng, 420, 2, 2, d)
    toward(q, k, np.arange(420), step * 4 * (np.arange(420) // 16))
    packed_case(ctx, q, k, v, starts_of([420]))


@pytest.mark.parametrize("d", DIMS)
def test_packed_rows_of_one_wave_with_references_apart(ctx, d):
    """Rows of a tile for which the far key is far above, far below or like the rest."""
    rng = np.random.default_rng(d)
    q, k, v = normal(rng, 260, 2, 1, d)
    toward(q, k, [100, 180], 30.0)
    q[::3, :, 0], q[1::3, :, 0] = -8, 0
    packed_case(ctx, q, k, v, starts_of([260]))


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("keys", [1500, 2500, 6000])
@pytest.mark.parametrize("where,score", [(0.02, 30.0), (0.5, 40.0), (0.97, 25.0), (0.5, -60.0)])
def test_paged_a_key_far_from_the_rest_in_one_piece(ctx, d, keys, where, score):
    """Pieces with references far apart, joined at once (1500 and 2500 keys) and in two steps."""
    rng = np.random.default_rng(d + keys)
    cache = Cache(ctx, rng, [keys, 90], keys // 16 + 1, 16, 1, d)
    starts = starts_of([9, 4])
    q = rng.standard_normal((13, 5, d)).astype(np.float16)
    toward(q, cache.rows[0][0], [int(where * keys)], score)
    toward(q, cache.rows[1][0], [60, 88], score)
    stored(cache)
    hold(paged(ctx, cache, q, starts, 5), *paged_want(cache, q, starts, True))


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("total", [100.0, -100.0])
def test_paged_scores_that_grow_from_piece_to_piece(ctx, d, total):
    rng = np.random.default_rng(d)
    keys = 6000
    cache = Cache(ctx, rng, [keys], keys // 16, 16, 2, d)
    starts = starts_of([40])
    q = rng.standard_normal((40, 4, d)).astype(np.float16)
    toward(q, cache.rows[0][0], np.arange(keys), total * (np.arange(keys) // 64) / 94)
    stored(cache)
    hold(paged(ctx, cache, q, starts, 4), *paged_want(cache, q, starts, True))


def test_row_starts_that_overlap_leave_nothing_behind(ctx):
    """More row tiles, and more pieces of them, than the rows can have by themselves: the rows behind
    stay as they are, and the call after it has its own results."""
    rng = np.random.default_rng(5)
    d, n, keys = 64, 1280, 20000
    cache = Cache(ctx, rng, [keys, 40, keys, 40, keys], keys // 16, 16, 1, d)
    q = rng.standard_normal((n + 2, 1, d)).astype(np.float16)
    got = paged(ctx, cache, q, np.array([0, n, 0, n, 0, n], np.uint32), 1)
    assert (got[n:] == 0x1234).all() and np.isfinite(got[:n].view(np.float16)).all()
    starts = starts_of([2, 0, 1, 1, 1])
    hold(paged(ctx, cache, q[:5], starts, 1), *paged_want(cache, q[:5], starts, True))
