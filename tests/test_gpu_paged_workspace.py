"""How much device memory the packed and paged calls lease: no more than what the call can use,
which a graph that holds one then keeps."""
from __future__ import annotations

import numpy as np
import pytest

import mi_attn
from mi_attn import U32, AttentionConfig

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def grown(kind, heads, d, rows, keys):
    """Bytes by which a new context's memory grows over one call."""
    hq, hkv = heads
    with mi_attn.Context(0) as ctx:
        q, out = ctx.empty((rows, hq, d)), ctx.empty((rows, hq, d))
        k = ctx.empty((rows, hkv, d))
        starts = ctx.tensor(np.array([0, rows], np.uint32), U32)
        width = max(1, -(-keys // 16))
        pages = ctx.empty((1, 16, hkv, d))
        table = ctx.tensor(np.full((1, width), 9, np.uint32), U32)  # no page: no key is read
        lengths = ctx.tensor(np.array([keys], np.uint32), U32)
        before = ctx.allocated_bytes()
        batch = ctx.begin_batch()
        if kind == "packed":
            batch.attention_packed(q, k, k, starts, AttentionConfig(hq, hkv, d), out=out)
        else:
            batch.attention_paged(q, pages, pages, table, lengths, starts, AttentionConfig(hq, hkv, d), out=out)
        batch.finish()
        return ctx.allocated_bytes() - before


@pytest.mark.parametrize("kind,heads,d,rows,keys,most", [
    ("packed", (16, 8), 128, 900, 0, 0),            # 15 key tiles: none is cut
    ("packed", (16, 8), 256, 450, 0, 0),
    ("packed", (16, 8), 128, 1, 0, 0),
    ("paged", (16, 8), 128, 1, 900, 0),
    ("paged", (16, 8), 128, 1, 100_000, 32),        # one row tile of each KV head
    ("paged", (16, 8), 64, 1, 2000, 32),
    ("paged", (16, 8), 128, 3000, 20_000, 72),      # as much as a call takes
    ("paged", (16, 8), 256, 3000, 20_000, 72),
    ("paged", (1030, 1030), 128, 2, 5000, 72),
    ("paged", (512, 512), 128, 2, 5000, 72),
    ("paged", (300, 300), 256, 2, 5000, 72)])
def test_workspace(kind, heads, d, rows, keys, most):
    bytes_ = grown(kind, heads, d, rows, keys)
    assert bytes_ <= most * MIB, f"{bytes_ / MIB:.1f} MiB"
