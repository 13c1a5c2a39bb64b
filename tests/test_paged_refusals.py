"""CPU tests of what the packed and paged calls refuse. Their checks of tensors come
before the batch's, so a null batch reaches every one of them without a GPU: a call whose
tensors pass ends with "null batch"."""
from __future__ import annotations

import ctypes

import pytest

import mi_attn
from mi_attn import F16, F32, U32, AttentionConfig, MiError, QkNormRopeCacheConfig, describe

FAKE = 0x7F0000000000  # 256-B aligned; the checks never dereference it


def tensor(shape, dtype=F16, strides=None, offset=0):
    return mi_attn.Tensor(describe(FAKE + offset, shape, strides, dtype))


def good(op, hq=8, hkv=2, d=128, rows=5, sequences=3, size=16, pages=7, width=4):
    """Arguments that pass, by name."""
    a = dict(q=tensor((rows, hq, d)), k=tensor((rows, hkv, d)), v=tensor((rows, hkv, d)),
             q_weight=tensor((d,)), k_weight=tensor((d,)),
             key_pages=tensor((pages, size, hkv, d), strides=(hkv * size * d, d, size * d, 1)),
             value_pages=tensor((pages, size, hkv, d)), table=tensor((sequences, width), U32),
             lengths=tensor((sequences,), U32), row_starts=tensor((sequences + 1,), U32),
             config=AttentionConfig(hq, hkv, d), rope=QkNormRopeCacheConfig(0, 1e6, 1e-6),
             out=tensor((rows, hq, d)))
    if op == "decode":
        a["q"], a["out"] = tensor((sequences, hq, d)), tensor((sequences, hq, d))
    return a


ORDER = {
    "append": ("mi_qk_norm_rope_paged", ("q", "k", "v", "q_weight", "k_weight", "key_pages", "value_pages", "table",
                                         "lengths", "row_starts", "rope", "out")),
    "decode": ("mi_attention_decode_paged", ("q", "key_pages", "value_pages", "table", "lengths", "config", "out")),
    "packed": ("mi_attention_packed", ("q", "k", "v", "row_starts", "config", "out")),
    "paged": ("mi_attention_paged", ("q", "key_pages", "value_pages", "table", "lengths", "row_starts", "config",
                                     "out")),
}


def call(op, args):
    name, order = ORDER[op]
    values = [args[k] for k in order]
    status = getattr(mi_attn.lib(), name)(None, *[
        None if v is None else ctypes.byref(v.desc if isinstance(v, mi_attn.Tensor) else v) for v in values])
    if status:
        raise MiError(status, mi_attn.lib().mi_last_error().decode())


def refuse(op, status, fragment, **change):
    with pytest.raises(MiError) as err:
        call(op, {**good(op), **change})
    assert err.value.name == status, err.value
    assert fragment in err.value.message


@pytest.mark.parametrize("op", list(ORDER))
def test_what_passes_reaches_the_batch(op):
    for hq, hkv, d, size in ((8, 2, 128, 16), (7, 7, 32, 64), (12, 4, 64, 1024), (48, 1, 256, 32)):
        args = good(op, hq, hkv, d, size=size)
        with pytest.raises(MiError) as err:
            call(op, args)
        assert err.value.name == "MI_ERR_INVALID_ARGUMENT" and err.value.message == "null batch"


@pytest.mark.parametrize("op", list(ORDER))
def test_null_tensors(op):
    for name in ORDER[op][1]:
        if op == "append" and name == "row_starts":
            continue
        fragment = "both weights, or none" if name.endswith("weight") else "null tensor or config"
        refuse(op, "MI_ERR_INVALID_ARGUMENT", fragment, **{name: None})
    refuse(op, "MI_ERR_INVALID_ARGUMENT", "query has no data", q=mi_attn.Tensor(describe(0, (3, 8, 128))))


def test_append_without_norm_or_row_starts():
    args = good("append", rows=3)
    args.update(q_weight=None, k_weight=None, row_starts=None)
    with pytest.raises(MiError, match="null batch"):
        call("append", args)
    # One row per sequence: the table and the lengths are of as many sequences.
    refuse("append", "MI_ERR_SHAPE", "block table must be", row_starts=None)


@pytest.mark.parametrize("op", list(ORDER))
def test_types_and_ranks(op):
    names = [n for n in ORDER[op][1] if n not in ("config", "rope")]
    for name in names:
        t = good(op)[name]
        wrong = F32 if t.dtype == F16 else F16
        refuse(op, "MI_ERR_DTYPE", "unsupported dtype", **{name: tensor(t.shape, wrong)})
        if len(t.shape) < 4:
            with pytest.raises(MiError) as err:
                call(op, {**good(op), name: tensor(t.shape + (1,), t.dtype)})
            assert err.value.name == "MI_ERR_SHAPE"


@pytest.mark.parametrize("op", list(ORDER))
def test_rows_that_the_kernels_cannot_read(op):
    n, hq, d = good(op)["q"].shape
    for name in ("q", "out"):
        refuse(op, "MI_ERR_SHAPE", "16-byte aligned rows", **{name: tensor((n, hq, d), offset=2)})
        refuse(op, "MI_ERR_SHAPE", "16-byte aligned rows", **{name: tensor((n, hq, d), strides=(hq * d + 4, d, 1))})
        refuse(op, "MI_ERR_SHAPE", "16-byte aligned rows", **{name: tensor((n, hq, d), strides=(hq * d, 1, hq))})
    if op != "packed":
        refuse(op, "MI_ERR_SHAPE", "position stride", key_pages=tensor((7, 16, 2, 128), strides=(4096, -256, 128, 1)))
        refuse(op, "MI_ERR_SHAPE", "position stride",
               value_pages=tensor((7, 16, 2, 128), strides=(4096, 1 << 27, 128, 1)))
    else:
        refuse(op, "MI_ERR_SHAPE", "row stride", k=tensor((5, 2, 128), strides=(-256, 128, 1)))
        refuse(op, "MI_ERR_SHAPE", "row stride", v=tensor((5, 2, 128), strides=(1 << 25, 128, 1)))


@pytest.mark.parametrize("op", ["decode", "packed", "paged"])
def test_heads_and_shapes(op):
    refuse(op, "MI_ERR_SHAPE", "do not match config", config=AttentionConfig(4, 2, 128))
    refuse(op, "MI_ERR_SHAPE", "do not match config", config=AttentionConfig(8, 4, 128))
    refuse(op, "MI_ERR_SHAPE", "divisible by kv_heads", config=AttentionConfig(8, 3, 128))
    refuse(op, "MI_ERR_SHAPE", "divisible by kv_heads", config=AttentionConfig(8, 0, 128))
    refuse(op, "MI_ERR_SHAPE", "query's shape", out=tensor((5, 8, 64)))
    for d in (16, 96, 512):
        args = good(op, d=d)
        with pytest.raises(MiError, match="head_dim must be 32, 64, 128, or 256"):
            call(op, args)


@pytest.mark.parametrize("op", ["append", "decode", "paged"])
def test_pages_tables_and_lengths(op):
    for size in (1, 8, 24, 48):
        with pytest.raises(MiError, match="power of two of at least 16"):
            call(op, good(op, size=size))
    refuse(op, "MI_ERR_SHAPE", "power of two", key_pages=tensor((0, 16, 2, 128)), value_pages=tensor((0, 16, 2, 128)))
    refuse(op, "MI_ERR_SHAPE", "same shape", value_pages=tensor((6, 16, 2, 128)))
    refuse(op, "MI_ERR_SHAPE", "block table must be", table=tensor((2, 4), U32))
    refuse(op, "MI_ERR_SHAPE", "block table must be", table=tensor((3, 0), U32))
    refuse(op, "MI_ERR_SHAPE", "unit innermost stride", table=tensor((3, 4), U32, strides=(1, 3)))
    refuse(op, "MI_ERR_SHAPE", "31 bits", table=tensor((3, 1 << 27), U32))
    refuse(op, "MI_ERR_SHAPE", "lengths must have 3 entries", lengths=tensor((4,), U32))
    refuse(op, "MI_ERR_SHAPE", "unit stride", lengths=tensor((3,), U32, strides=(2,)))


@pytest.mark.parametrize("op", ["append", "packed", "paged"])
def test_row_starts(op):
    refuse(op, "MI_ERR_SHAPE", "one entry more", row_starts=tensor((0,), U32))
    refuse(op, "MI_ERR_SHAPE", "unit stride", row_starts=tensor((4,), U32, strides=(2,)))
    if op != "packed":
        refuse(op, "MI_ERR_SHAPE", "block table must be", row_starts=tensor((5,), U32))


def test_append_shapes_and_theta():
    refuse("append", "MI_ERR_SHAPE", "incompatible", k=tensor((4, 2, 128)))
    refuse("append", "MI_ERR_SHAPE", "key's shape", v=tensor((5, 4, 128)))
    refuse("append", "MI_ERR_SHAPE", "incompatible", q_weight=tensor((64,)))
    refuse("append", "MI_ERR_SHAPE", "query's shape", out=tensor((5, 4, 128)))
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        refuse("append", "MI_ERR_SHAPE", "positive theta", rope=QkNormRopeCacheConfig(0, theta, 1e-6))


def test_packed_keys_are_of_the_querys_rows():
    refuse("packed", "MI_ERR_SHAPE", "do not match config", k=tensor((4, 2, 128)))
    refuse("packed", "MI_ERR_SHAPE", "do not match config", v=tensor((5, 4, 128)))


def test_launch_limits():
    big = tensor((1 << 24, 128, 128))
    for op, change in (("packed", dict(k=tensor((1 << 24, 1, 128)), v=tensor((1 << 24, 1, 128)))),
                       ("append", dict(k=tensor((1 << 24, 1, 128)), v=tensor((1 << 24, 1, 128)),
                                       key_pages=tensor((7, 16, 1, 128)), value_pages=tensor((7, 16, 1, 128))))):
        refuse(op, "MI_ERR_SHAPE", "launch limits", q=big, out=big, config=AttentionConfig(128, 1, 128), **change)
