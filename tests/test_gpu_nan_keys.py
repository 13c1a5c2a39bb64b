"""A piece or split whose keys are all NaN makes its rows NaN, as the same keys do in one part:
the merges tell it from one without a key."""
import numpy as np
import pytest

import mi_attn
from helpers import f16, oracle_attention, run_attention, upload_kv

pytestmark = pytest.mark.gpu
NAN = np.float16(np.nan).view(np.uint16)


def rand(seed, shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float16).view(np.uint16)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,cap,lengths", [
    (16, 8, 1300, [129, 257, 385, 700]),                         # pieces of 128 keys, the last of one
    (8, 1, 6000, [5889, 129, 40]),                               # 47 pieces: overflow slots
    (32, 8, 1200, [1025, 1153, 1121, 1057] * 6),                 # segments that end within the sequences
    (8, 8, 2100, [32 * n + 1 for n in range(1, 66)])])
def test_batched_decode_nan_in_the_newest_key(ctx, hq, hkv, d, cap, lengths):
    B = len(lengths)
    q, k, v = rand(1, (B, hq, d)), rand(2, (B, cap, hkv, d)), rand(3, (B, cap, hkv, d))
    for b, n in enumerate(lengths[:-1]):
        k[b, n - 1] = NAN
    kt, vt = (ctx.tensor(np.ascontiguousarray(x.transpose(0, 2, 1, 3))) for x in (k, v))
    views = [t.view(k.shape, (hkv * cap * d, d, cap * d, 1)) for t in (kt, vt)]
    lt = ctx.tensor(np.asarray(lengths, np.uint32), mi_attn.U32)
    batch = ctx.begin_batch()
    out = batch.attention_decode_batched(ctx.tensor(q), *views, lt, mi_attn.AttentionConfig(hq, hkv, d, True, 0))
    batch.finish()
    got = f16(ctx.download(out))
    for b, n in enumerate(lengths[:-1]):
        assert np.isnan(got[b]).all(), f"length {n}"
    n = lengths[-1]
    ref = oracle_attention(q[-1:], k[-1, :n], v[-1, :n], hq=hq, hkv=hkv, d=d, off=n - 1)["f32"]
    assert np.abs(got[-1:] - ref).max() <= 2e-3


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,off", [(24, 1100), (31, 20000), (300, 700)])
def test_tiled_nan_in_every_key_of_some_splits(ctx, d, T, off):
    hq, hkv, L = 8, 1, off + T
    q, k, v = rand(4, (T, hq, d)), rand(5, (L, hkv, d)), rand(6, (L, hkv, d))
    cfg = mi_attn.AttentionConfig(hq, hkv, d, True, off)
    _, view = upload_kv(ctx, k, "head_major")
    info = ctx.plan(ctx.tensor(q), view, view, cfg, mi_attn.TILED)
    assert info["kernel"] == "attn_tiled" and info["splits"] > 1, info
    block = info["block_keys"]
    k[block:2 * block] = NAN
    got = f16(run_attention(ctx, q, k, v, hq=hq, hkv=hkv, d=d, off=off, kind="tiled"))
    assert np.isnan(got).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["flash-decode", "decode-split-kv", "tiled"])
@pytest.mark.parametrize("L", [2049, 20001])
def test_one_token_nan_in_the_newest_keys(ctx, d, kind, L):
    """The other kernels of one token that split their keys: NaN from a tile's start to the end."""
    hq, hkv = 8, 2
    q, v = rand(7, (1, hq, d)), rand(9, (L, hkv, d))
    for first in (L - 1, L - 33, L - 129, L - 257, L - 1025):
        k = rand(8, (L, hkv, d))
        k[first:] = NAN
        got = f16(run_attention(ctx, q, k, v, hq=hq, hkv=hkv, d=d, off=L - 1, kind=kind))
        assert np.isnan(got).all(), f"from key {first}"
