"""The paged KV cache's operators and attention over packed sequences, as calls to time.

A server keeps the keys and values of all its sequences in one pool of pages and packs the new
tokens of a step into rows, sequence after sequence. `op` is the operator of a case:
  append   Q/K norm and RoPE of packed rows, K and V written into the pages of their sequences
  decode   attention of one new token per sequence over its pages
  packed   causal attention of whole prompts over their own packed rows of K and V
  paged    causal attention of packed new tokens over the pages of their sequences

Keys of a case: `batch` sequences; each has between t_low and t_high new rows on o_low to o_high
cached positions; q_heads / kv_heads heads of head_dim; pages of `page` positions; `norm`: whether
Q and K are normalised before the rotation. All tensors are f16, tables and lengths u32.

Sizes: the head counts that the repository is measured on (16/8, 32/8, 40/8 and 64/8), and others
that its tests use; head dimensions 32 to 256; sequences of one token to tens of thousands.
"""
import sys
from pathlib import Path

import numpy as np
import torch

own = False

THETA, EPS = 1_000_000.0, 1e-6
HEADS = [(16, 8), (32, 8), (40, 8), (64, 8), (32, 8), (8, 1), (12, 4), (7, 7)]
PAGES = [16, 16, 32, 64, 128, 256]


def _case(name, op, batch, rows, cached, heads, head_dim, page, norm=True):
    return dict(name=name, op=op, batch=batch, t_low=rows[0], t_high=rows[1], o_low=cached[0], o_high=cached[1],
                q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim, page=page, norm=norm)


def listed():
    return [
        # The next token of a lightly loaded server on the smallest model: latency.
        _case("append 8x1 16/8", "append", 8, (1, 1), (39, 999), (16, 8), 128, 16),
        # Nine prompts of a step, for a model without Q/K norm.
        _case("append 9x3-900 32/8/64", "append", 9, (3, 900), (0, 0), (32, 8), 64, 32, False),
        # Chunks of four long documents, the largest heads, far positions.
        _case("append 4x2048 64/8", "append", 4, (2048, 2048), (0, 60000), (64, 8), 128, 64),
        # The next token of a lightly loaded server on the smallest model: latency.
        _case("decode 8 16/8 L40-1000", "decode", 8, (1, 1), (39, 999), (16, 8), 128, 16),
        # The repository's headline, through pages: 32 sequences of 1024 to 8192 tokens.
        _case("decode 32 32/8 L1024-8192", "decode", 32, (1, 1), (1023, 8191), (32, 8), 128, 64),
        # Many sequences at the other common head dimension.
        _case("decode 70 32/8/64 L100-4000", "decode", 70, (1, 1), (99, 3999), (32, 8), 64, 16),
        # Short questions that arrive together, the smallest model.
        _case("packed 12x3-130 16/8", "packed", 12, (3, 130), (0, 0), (16, 8), 128, 16),
        # Prompts of a few paragraphs, groups of 5.
        _case("packed 7x150-1500 40/8", "packed", 7, (150, 1500), (0, 0), (40, 8), 128, 16),
        # Two long prompts.
        _case("packed 2x4000-6000 32/8", "packed", 2, (4000, 6000), (0, 0), (32, 8), 128, 16),
        # Chats' next questions, a few tokens each on cached conversations.
        _case("paged 16x2-40@200-6000 32/8", "paged", 16, (2, 40), (200, 6000), (32, 8), 128, 16),
        # A mixed step at the largest head dimension.
        _case("paged 5x1-300@0-2000 16/4/256", "paged", 5, (1, 300), (0, 2000), (16, 4), 256, 32),
        # A chunk of a long document, the largest heads.
        _case("paged 1x2048@16384 64/8", "paged", 1, (2048, 2048), (16384, 16384), (64, 8), 128, 256),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return max(low, min(high, int(low * (high / low) ** rng.random() + rng.random())))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "packed", "paged", "paged"])
    heads, d = rng.choice(HEADS), rng.choice([128, 128, 128, 64, 64, 32, 256])
    c = _case("", op, 1, (1, 1), (0, 0), heads, d, rng.choice(PAGES), rng.random() < 0.7)
    if op == "decode":
        c["batch"] = _spread(rng, 1, 128)
        c["o_high"] = _spread(rng, 1, min(60000, 300_000 // c["batch"]))
        c["o_low"] = int(c["o_high"] * rng.random())
    else:
        c["batch"] = _spread(rng, 1, 48)
        c["t_high"] = _spread(rng, 2, min(3000, 16000 // c["batch"]))
        c["t_low"] = rng.choice([1, max(1, int(c["t_high"] * rng.random()))])
        if op != "packed" and rng.random() < 0.8:
            c["o_high"] = _spread(rng, 8, min(20000, 100_000 // c["batch"]))
            c["o_low"] = int(c["o_high"] * rng.random())
    # No more than the largest listed case: products, and the scores that a plain form holds.
    while work(c)["flops"] > 8e11 or _most_scores(c) > 2e9:
        c["t_high"] = max(1, c["t_high"] * 2 // 3)
        c["t_low"] = min(c["t_low"], c["t_high"])
    del c["name"]
    return c


def _most_scores(c):
    return c["batch"] * c["q_heads"] * c["t_high"] * (c["o_high"] + c["t_high"]) if c["op"] != "append" else 0


# ------------------------------------------------------------------- inputs --

def _ragged(r, n, low, high):
    """n whole numbers from low to high, of the mean between them: any seed is the same work."""
    a = r.integers(low, high + 1, n)
    left = n * (low + high) // 2 - int(a.sum())
    for i in range(n):
        step = min(max(left, low - int(a[i])), high - int(a[i]))
        a[i] += step
        left -= step
    return r.permutation(a)


def _sizes(case, seed):
    """New rows and cached positions of each sequence."""
    r = np.random.default_rng(seed % (1 << 32))
    n = case["batch"]
    return _ragged(r, n, case["t_low"], case["t_high"]), _ragged(r, n, case["o_low"], case["o_high"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, cached = _sizes(case, seed)
    hq, hkv, d, s, b = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page", "batch"))
    n = int(rows.sum())

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16).mul_(scale)

    def words(a):
        return torch.from_numpy(np.asarray(a).astype(np.int32)).cuda()

    state = dict(op=case["op"], row_starts=words(np.concatenate([[0], np.cumsum(rows)])), lengths=words(rows + cached),
                 most_rows=case["t_high"], one_row=case["t_high"] == 1, out=torch.empty(n, hq, d, device="cuda", dtype=torch.float16))
    if case["op"] in ("append", "packed"):
        # The rows of a fused QKV projection, as a model hands them over.
        qkv = normal(n, hq + 2 * hkv, d)
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
    else:
        state["q"] = normal(n, hq, d, scale=1.5)
    if case["op"] == "append":
        state["weights"] = [torch.rand(d, generator=g, device="cuda").mul_(1.5).add_(0.5).half() for _ in "qk"] if case["norm"] else None
    if case["op"] != "packed":
        # Pages in the order in which a busy pool hands them out; the table's tail holds no page.
        width = -(-(case["o_high"] + case["t_high"]) // s)
        used = -(-(rows + cached) // s)
        pages = b * width + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((b, width), -1, device="cuda", dtype=torch.int32)
        for i, first in enumerate(np.concatenate([[0], np.cumsum(used)[:-1]])):
            table[i, :used[i]] = order[first:first + used[i]]
        # [pages, KV heads, positions, head_dim], seen as [pages, positions, KV heads, head_dim].
        state.update(table=table, key_pages=normal(pages, hkv, s, d).transpose(1, 2),
                     value_pages=normal(pages, hkv, s, d).transpose(1, 2))
    torch.cuda.synchronize()  # the inputs were made on torch's stream; a user's calls may run on another
    return state


# -------------------------------------------------------------- plain forms --

def _places(x):
    """Of each packed row: its sequence, its place among the sequence's new rows, its position."""
    starts = x["row_starts"].long()
    row = torch.arange(x["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return seq, row - starts[seq], x["lengths"].long()[seq] - starts[seq + 1] + row


def _rotated(x, weight, position):
    x = x.float()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    half = x.shape[-1] // 2
    # Angles of far positions lose their fraction in 32 bits.
    turn = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = position.double()[:, None, None] * turn
    c, s = angle.cos().float(), angle.sin().float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, a * s + b * c], -1).half()


def _plain_append(x):
    seq, _, position = _places(x)
    qw, kw = x["weights"] or (None, None)
    size = x["key_pages"].shape[1]
    page = x["table"].long()[seq, position // size]
    x["key_pages"][page, position % size] = _rotated(x["k"], kw, position)
    x["value_pages"][page, position % size] = x["v"]
    return {"q": _rotated(x["q"], qw, position), "key_pages": x["key_pages"], "value_pages": x["value_pages"]}


def _plain_attention(x):
    seq, place, _ = _places(x)
    starts, n = x["row_starts"].long(), x["q"].shape[0]
    hq, d = x["q"].shape[1:]
    b, t = starts.shape[0] - 1, x["most_rows"]
    at = (starts[:-1, None] + torch.arange(t, device="cuda")).clamp(max=n - 1)
    if x["op"] == "packed":
        key, value = x["k"][at], x["v"][at]
        lengths = starts[1:] - starts[:-1]
    else:
        table = x["table"].long()
        key, value = (p[table].flatten(1, 2) for p in (x["key_pages"], x["value_pages"]))
        lengths = x["lengths"].long()
    hkv = key.shape[2]
    # [B, KV heads, group x rows, D] by [B, KV heads, D, keys].
    q = x["q"][at].float().view(b, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    score = torch.matmul(q * d ** -0.5, key.float().permute(0, 2, 3, 1))
    last = (lengths - (starts[1:] - starts[:-1]))[:, None] + torch.arange(t, device="cuda")
    unseen = torch.arange(key.shape[1], device="cuda") > last[:, :, None]
    score = score.view(b, hkv, hq // hkv, t, -1).masked_fill_(unseen[:, None, None], float("-inf"))
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    weight = weight.div_(weight.sum(-1, keepdim=True)).view(b, hkv, (hq // hkv) * t, -1)
    out = torch.matmul(weight, value.float().transpose(1, 2))
    return out.view(b, hkv, hq // hkv, t, d).permute(0, 3, 1, 2, 4)[seq, place].reshape(n, hq, d).half()


# ------------------------------------------------------ the framework's calls --

_program = {"passes": 0, "batch": None, "before": None, "context": None}


def _batch():
    """The program's open batch: one for every 32 operators, as for the layers of a forward pass,
    and at most two in flight."""
    p = _program
    if p["passes"] % 32 == 0:
        if p["before"] is not None:
            p["before"].wait()
        p["before"] = p["batch"].commit() if p["batch"] is not None else None
        p["batch"] = p["context"].begin_batch()
    p["passes"] += 1
    return p["batch"]


def _views(x):
    """The tensors of a state as the framework's descriptors, which a program makes once: the
    state's tensors may be filled anew between passes but not replaced, and are held here, as a
    descriptor does not keep its memory alive."""
    if _program["context"] is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "metal-infer-rs_amd"))
    import mi_attn

    if _program["context"] is None:
        _program["context"] = mi_attn.Context(torch.cuda.current_device())

    def view(t):
        if t is None:
            return None
        kind = mi_attn.U32 if t.dtype == torch.int32 else mi_attn.F16
        return mi_attn.Tensor(mi_attn.describe(t.data_ptr(), tuple(t.shape), tuple(t.stride()), kind))

    names = ("q", "k", "v", "out", "table", "lengths", "row_starts", "key_pages", "value_pages")
    w = {k: view(x.get(k)) for k in names}
    w["q_weight"], w["k_weight"] = (view(t) for t in x.get("weights") or (None, None))
    w["held"] = [x.get(k) for k in (*names, "weights")]
    hkv = (x["k"] if x["op"] in ("append", "packed") else x["key_pages"]).shape[-2]
    w["attention"] = mi_attn.AttentionConfig(x["q"].shape[1], hkv, x["q"].shape[2], True, 0)
    w["rope"] = mi_attn.QkNormRopeCacheConfig(0, THETA, EPS)
    return w


def _own(x):
    """Enqueues on the context's stream, which torch's streams do not wait for: the caller waits
    for the device before it reads the outputs, fills the inputs anew or drops the state."""
    if "views" not in x:
        x["views"] = _views(x)
    w, batch = x["views"], _batch()
    if x["op"] == "append":
        batch.qk_norm_rope_paged(w["q"], w["k"], w["v"], w["q_weight"], w["k_weight"], w["key_pages"], w["value_pages"],
                                 w["table"], w["lengths"], w["rope"], row_starts=None if x["one_row"] else w["row_starts"],
                                 out=w["out"])
        return {"q": x["out"], "key_pages": x["key_pages"], "value_pages": x["value_pages"]}
    if x["op"] == "decode":
        batch.attention_decode_paged(w["q"], w["key_pages"], w["value_pages"], w["table"], w["lengths"],
                                     w["attention"], out=w["out"])
    elif x["op"] == "packed":
        batch.attention_packed(w["q"], w["k"], w["v"], w["row_starts"], w["attention"], out=w["out"])
    else:
        batch.attention_paged(w["q"], w["key_pages"], w["value_pages"], w["table"], w["lengths"], w["row_starts"],
                              w["attention"], out=w["out"])
    return x["out"]


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["op"] == "append" else _plain_attention(state)


# ------------------------------------------------------- work and exactness --

def work(case):
    hq, hkv, d = (case[k] for k in ("q_heads", "kv_heads", "head_dim"))
    tl, th, b = case["t_low"], case["t_high"], case["batch"]
    t, o = (tl + th) / 2, (case["o_low"] + case["o_high"]) / 2
    square = (tl * tl + tl * th + th * th) / 3
    if case["op"] == "append":
        # Q read and written, K and V read and written; two products and a sum per rotated value.
        return {"bytes": 2 * b * t * d * (2 * hq + 4 * hkv), "flops": (8 if case["norm"] else 3) * b * t * d * (hq + hkv)}
    pairs = b * (t * o + (square + t) / 2)
    return {"bytes": 2 * b * d * (2 * t * hq + 2 * (o + t) * hkv), "flops": 4 * d * hq * pairs}


def exact(case, seed):
    x = prepare(case, seed)
    rows, cached = _sizes(case, seed)
    first = np.concatenate([[0], np.cumsum(rows)])
    hq, hkv, d, size = (case[k] for k in ("q_heads", "kv_heads", "head_dim", "page"))
    q = x["q"].double()
    out = torch.empty_like(q)
    if case["op"] == "append":
        keys, values = x["key_pages"].double(), x["value_pages"].double()
        powers = torch.arange(d // 2, device="cuda", dtype=torch.float64) * (-2.0 / d)
        turns = torch.exp(powers * float(np.log(THETA)))
        for i in range(case["batch"]):
            at = slice(int(first[i]), int(first[i + 1]))
            where = int(cached[i]) + torch.arange(int(rows[i]), device="cuda")
            pages = x["table"][i, where // size].long()
            wave = torch.polar(torch.ones(1, device="cuda", dtype=torch.float64), where[:, None].double() * turns)[:, None]
            for name, index in (("q", 0), ("k", 1)):
                y = x[name][at].double()
                if x["weights"] is not None:
                    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * x["weights"][index].double()
                z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * wave
                y = torch.cat([z.real, z.imag], -1)
                if name == "q":
                    out[at] = y
                else:
                    keys[pages, where % size] = y
            values[pages, where % size] = x["v"][at].double()
        return {"q": out, "key_pages": keys, "value_pages": values}
    for i in range(case["batch"]):
        total = int(rows[i] + cached[i])
        lo, hi = int(first[i]), int(first[i + 1])
        if case["op"] == "packed":
            k, v, total = x["k"][lo:hi], x["v"][lo:hi], hi - lo
        else:
            pages = x["table"][i, :-(-total // size)].long()
            k, v = (x[p][pages].reshape(-1, hkv, d)[:total] for p in ("key_pages", "value_pages"))
        for h in range(hkv):
            kd, vd = k[:, h].double(), v[:, h].double()
            step = max(1, int(5e7 // (total * (hq // hkv))))
            for a in range(lo, hi, step):
                e = min(hi, a + step)
                part = q[a:e, h * (hq // hkv):(h + 1) * (hq // hkv)]
                s = (part.reshape(-1, d) @ kd.T / d ** 0.5).view(e - a, -1, total)
                position = total - (hi - lo) + torch.arange(a - lo, e - lo, device="cuda")
                s = s + torch.where(torch.arange(total, device="cuda")[None] <= position[:, None], 0.0, -torch.inf)[:, None]
                p = torch.softmax(s, -1).view(-1, total)
                out[a:e, h * (hq // hkv):(h + 1) * (hq // hkv)] = (p @ vd).view(part.shape)
    return out
