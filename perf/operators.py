"""The operators of a decode step over a paged key-value cache, and the calls that are measured.

Three kinds of work:

  w4      a linear layer of a few rows with 4-bit weights and group scales (``lib.pack_w4``, ``lib.matmul_w4``): the projections
          around the attention of new tokens
  append  new keys and values into a paged cache, with the rotation of their positions and of the queries' on the way
          (``lib.paged_kv_append``): single tokens and prompts
  attend  attention of one new token per sequence over the paged cache (``lib.paged_attention``)

With ``own`` false, ``run`` computes the same in elementary torch operations in 32 bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def _lib():
    path = os.path.abspath("graph-compiler_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gc_b200 import lib

    return lib


# ----------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest attention call: one conversation of about a thousand tokens, the head layout of a grouped-query decoder
        {"name": "attend_one", "kind": "attend", "sequences": 1, "heads": 32, "kv_heads": 8, "dim": 128, "length": 1031, "spread": "same", "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16", "layout": "heads"},
        # an ordinary serving batch: conversations of all lengths up to four thousand tokens
        {"name": "attend_batch", "kind": "attend", "sequences": 64, "heads": 32, "kv_heads": 8, "dim": 128, "length": 4096, "spread": "ragged", "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16", "layout": "heads"},
        # a key head to each query head (the head layout of this repository's llama2 partitions), f16, tokens outside heads
        {"name": "attend_heads", "kind": "attend", "sequences": 16, "heads": 32, "kv_heads": 32, "dim": 128, "length": 2048, "spread": "same", "page": 32, "window": 0, "dtype": "f16", "cache": "f16", "layout": "tokens"},
        # one long document: all the work is in two sequences' length
        {"name": "attend_long", "kind": "attend", "sequences": 2, "heads": 64, "kv_heads": 8, "dim": 128, "length": 131071, "spread": "same", "page": 64, "window": 0, "dtype": "bf16", "cache": "bf16", "layout": "heads"},
        # the largest: a full batch over a cache held in 8 bits
        {"name": "attend_8bit", "kind": "attend", "sequences": 128, "heads": 64, "kv_heads": 8, "dim": 128, "length": 8192, "spread": "ragged", "page": 64, "window": 0, "dtype": "bf16", "cache": "e4m3", "layout": "heads"},
        # odd everything: seven query heads to a key head, short heads, pages that are no power of two, a window, idle sequences
        {"name": "attend_odd", "kind": "attend", "sequences": 37, "heads": 28, "kv_heads": 4, "dim": 80, "length": 1999, "spread": "skewed", "page": 24, "window": 700, "dtype": "f16", "cache": "f16", "layout": "tokens"},
        # one new token of each of 64 conversations
        {"name": "append_step", "kind": "append", "sequences": 64, "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "reach": 32768, "page": 16, "dtype": "bf16", "cache": "bf16", "layout": "heads"},
        # prompts of mixed lengths, 8192 tokens in all
        {"name": "append_prompts", "kind": "append", "sequences": 5, "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "reach": 4096, "page": 16, "dtype": "bf16", "cache": "bf16", "layout": "heads"},
        # pieces of prompts far into long documents, an 8-bit cache, neighbouring pairs of half a head rotated
        {"name": "append_8bit", "kind": "append", "sequences": 7, "tokens": 3001, "heads": 28, "kv_heads": 4, "dim": 80, "rotary": 40, "interleaved": True, "reach": 1000000, "page": 24, "dtype": "f16", "cache": "e4m3", "layout": "tokens"},
        # one token through a projection of the decoder block
        {"name": "w4_one", "kind": "w4", "M": 1, "N": 4096, "K": 4096, "group": 128, "zeros": False, "bias": False, "relu": False, "dtype": "bf16"},
        # a batch of sixteen through the largest decode-shaped layer of the benchmark
        {"name": "w4_wide", "kind": "w4", "M": 16, "N": 28672, "K": 8192, "group": 128, "zeros": False, "bias": False, "relu": False, "dtype": "bf16"},
        # five rows, an odd number of outputs, zero points and small groups
        {"name": "w4_odd", "kind": "w4", "M": 5, "N": 11001, "K": 4095, "group": 32, "zeros": True, "bias": True, "relu": True, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attend(rng):
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16] if kv_heads <= 8 else [1, 2])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3"])
    sequences, length = _log(rng, 1, 256), _log(rng, 1, 131072)
    while sequences * length * kv_heads * dim * (1 if cache == "e4m3" else 2) > 128 * 8192 * 8 * 128:
        sequences, length = max(1, sequences // 2), length if sequences > 1 else length // 2
    return {"kind": "attend", "sequences": sequences, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "length": length,
            "spread": rng.choice(["same", "ragged", "ragged", "skewed"]), "page": rng.choice([8, 16, 16, 24, 32, 64, 128]),
            "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "dtype": dtype, "cache": cache, "layout": rng.choice(["heads", "tokens"])}


def _draw_append(rng):
    dim = rng.choice([64, 80, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
    group = rng.choice([1, 2, 4, 4, 5, 7, 8, 16] if kv_heads <= 8 else [1, 2])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    tokens = _log(rng, 1, 8192)
    while tokens * kv_heads * (group + 2) * dim > 2 * 8192 * 48 * 128:
        tokens //= 2
    sequences = tokens if rng.random() < 0.5 and tokens <= 256 else min(tokens, _log(rng, 1, 64))
    return {"kind": "append", "sequences": sequences, "tokens": tokens, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "rotary": dim if rng.random() < 0.7 else dim // 2, "interleaved": rng.random() < 0.3, "reach": _log(rng, 1, 1000000) + tokens,
            "page": rng.choice([8, 16, 16, 24, 32, 64, 128]), "dtype": dtype, "cache": rng.choice([dtype, dtype, "e4m3"]), "layout": rng.choice(["heads", "tokens"])}


def _draw_w4(rng):
    m, n, k = _log(rng, 1, 16), _log(rng, 64, 28672), _log(rng, 64, 16384)
    grain = rng.choice(["tile", "tile", "eight", "odd"])
    if grain != "odd":
        step = 128 if grain == "tile" else 8
        n, k = max(step, n // step * step), max(step, k // step * step)
    while n * k > 28672 * 8192:
        n //= 2
    return {"kind": "w4", "M": m, "N": n, "K": k, "group": rng.choice([32, 64, 128, 128, 256]), "zeros": rng.random() < 0.4,
            "bias": rng.random() < 0.4, "relu": rng.random() < 0.2, "dtype": rng.choice(["bf16", "bf16", "f16"])}


def draw(rng):
    return rng.choice([_draw_attend, _draw_attend, _draw_append, _draw_w4, _draw_w4])(rng)


# ----------------------------------------------------------------------------- inputs
def _lengths(c):
    """Tokens in the cache of each sequence, by the case alone."""
    r, n, top = random.Random(c["sequences"] * 1000003 + c["length"]), c["sequences"], c["length"]
    if c["spread"] == "same":
        return [top] * n
    if c["spread"] == "ragged":
        got = [r.randint(max(1, top // 8), top) for _ in range(n)]
    else:   # most are short, a few long, some slots of the batch idle
        got = [0 if r.random() < 0.1 else _log(r, 1, top) for _ in range(n)]
    got[r.randrange(n)] = top
    return got


def _tokens(c):
    """(sequence, position) of each new token, by the case alone: whole numbers, tokens of one sequence together."""
    r, n, t = random.Random(c["sequences"] * 1000003 + c["tokens"]), c["sequences"], c["tokens"]
    cuts = sorted(r.sample(range(1, t), n - 1)) if n < t else list(range(1, t))
    counts = np.diff([0] + cuts + [t])
    starts = np.array([r.randint(0, max(0, c["reach"] - int(k))) for k in counts])
    seq = np.repeat(np.arange(n), counts)
    at = np.arange(t) - np.repeat(np.cumsum(counts) - counts, counts)
    return seq, np.repeat(starts, counts) + at


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, dtype, *shape, std=1.0):
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float16 if dtype in (torch.float16, torch.float8_e4m3fn) else dtype)
    return x.mul_(std).to(dtype)


def _pool(g, c, pages):
    """A cache of `pages` pages as [page, head, token, dim], whatever lies outside in memory; 8-bit codes of both signs and all sizes."""
    shape = (pages, c["kv_heads"], c["page"], c["dim"]) if c["layout"] == "heads" else (pages, c["page"], c["kv_heads"], c["dim"])
    x = _normal(g, DTYPES[c["cache"]], *shape, std=30.0 if c["cache"] == "e4m3" else 1.0)
    return x if c["layout"] == "heads" else x.transpose(1, 2)


def _scales(g, c):
    if c["cache"] != "e4m3":
        return None
    return (0.5 + torch.rand(c["kv_heads"], generator=g, device=DEV)) / 30.0


def _inputs_attend(c, g):
    lengths = _lengths(c)
    per = max(1, -(-c["length"] // c["page"]))
    pages = c["sequences"] * per
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(c["sequences"], per)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    used = torch.arange(per, device=DEV)[None] * c["page"] < lens[:, None]
    table = torch.where(used, table, torch.full_like(table, -1))
    return {"c": c, "q": _normal(g, DTYPES[c["dtype"]], c["sequences"], c["heads"], c["dim"], std=1.5), "keys": _pool(g, c, pages), "values": _pool(g, c, pages),
            "key_scale": _scales(g, c), "value_scale": _scales(g, c), "table": table, "lengths": lens, "scale": c["dim"] ** -0.5}


def _inputs_append(c, g):
    seq, pos = _tokens(c)
    page = c["page"]
    per = int(pos.max()) // page + 1
    table = np.full((c["sequences"], per), -1, dtype=np.int32)
    touched = np.unique(seq.astype(np.int64) * per + pos // page)
    pages = len(touched) + 3
    order = torch.randperm(pages, generator=g, device=DEV).cpu().numpy()
    table.reshape(-1)[touched] = order[: len(touched)]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    qkv = _normal(g, DTYPES[c["dtype"]], c["tokens"], (h + 2 * kv) * d)   # what a fused projection leaves: q, k and v are views of its rows
    q, k, v = qkv.split([h * d, kv * d, kv * d], dim=1)
    inv = 1.0 / 10000.0 ** (torch.arange(0, c["rotary"], 2, dtype=torch.float64, device=DEV) / c["rotary"])
    return {"c": c, "q": q.view(-1, h, d), "k": k.view(-1, kv, d), "v": v.view(-1, kv, d), "keys": _pool(g, c, pages), "values": _pool(g, c, pages),
            "key_scale": _scales(g, c), "value_scale": _scales(g, c), "table": torch.from_numpy(table).to(DEV), "inv_freq": inv,
            "seq": torch.from_numpy(seq.astype(np.int32)).to(DEV), "pos": torch.from_numpy(pos.astype(np.int32)).to(DEV)}


def _inputs_w4(c, g):
    n, k, dt = c["N"], c["K"], DTYPES[c["dtype"]]
    groups = -(-k // c["group"])
    return {"c": c, "x": _normal(g, dt, c["M"], k), "codes": torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8),
            "scales": ((0.5 + torch.rand(n, groups, generator=g, device=DEV)) * (0.2 * k ** -0.5)).to(dt),
            "zeros": torch.randint(0, 16, (n, groups), generator=g, device=DEV, dtype=torch.uint8) if c["zeros"] else None,
            "bias": _normal(g, dt, n, std=0.1) if c["bias"] else None}


def _inputs(c, seed):
    return {"attend": _inputs_attend, "append": _inputs_append, "w4": _inputs_w4}[c["kind"]](c, _gen(seed))


def prepare(case, seed):
    s, c = _inputs(case, seed), case
    if c["kind"] == "w4":
        s["out"] = torch.empty(c["M"], c["N"], dtype=DTYPES[c["dtype"]], device=DEV)
        if own:   # a program packs its weights once, when it loads them
            s["packed"] = _lib().pack_w4(s["codes"], s["scales"], c["K"], c["group"], zeros=s["zeros"])
    else:
        s["out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
        if own and c["kind"] == "attend":   # scratch memory that a program keeps beside its cache
            s["workspace"] = _lib().paged_attention_workspace(s["q"], s["keys"])
    return s


# ----------------------------------------------------------------------------- one pass
def _of_cache(cache, scale, table):
    """Keys or values as [sequence, head, token, dim] in 32 bits."""
    x = cache[table.clamp(min=0).long()].float()                      # [sequence, page, head, token, dim]
    if scale is not None:
        x = x * scale.view(1, 1, -1, 1, 1)
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    c, lens = s["c"], s["lengths"].view(-1, 1, 1, 1)
    b, kv = c["sequences"], c["kv_heads"]
    keys = _of_cache(s["keys"], s["key_scale"], s["table"])
    scores = (s["q"].float() * s["scale"]).view(b, kv, -1, c["dim"]) @ keys.transpose(2, 3)
    del keys
    at = torch.arange(scores.shape[-1], device=scores.device)
    seen = at < lens
    if c["window"]:
        seen = seen & (at >= lens - c["window"])
    scores = scores.masked_fill(~seen, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    out = (p @ _of_cache(s["values"], s["value_scale"], s["table"])) / total
    return torch.where(lens > 0, out, torch.zeros_like(out)).view(b, c["heads"], c["dim"]).to(s["q"].dtype)


def _rotate(x, cos, sin, c):
    r = c["rotary"]
    x, rest = x.float()[..., :r], x.float()[..., r:]
    if c["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        x = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2:]
        x = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([x, rest], dim=-1)


def _held(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x / scale.view(1, -1, 1)).clamp(-448.0, 448.0).to(dtype)


def _append(s):
    c, pos = s["c"], s["pos"].long()
    angle = s["pos"].double()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q, k = _rotate(s["q"], cos, sin, c), _rotate(s["k"], cos, sin, c)
    page, at = s["table"][s["seq"].long(), pos // c["page"]].long(), pos % c["page"]
    raw = lambda t: t.view(torch.uint8) if c["cache"] == "e4m3" else t  # noqa: E731
    raw(s["keys"])[page, :, at] = raw(_held(k, s["key_scale"], s["keys"].dtype))
    raw(s["values"])[page, :, at] = raw(_held(s["v"].float(), s["value_scale"], s["values"].dtype))
    return {"q": q.to(s["q"].dtype), "keys": s["keys"], "values": s["values"]}


def _w4(s):
    c, codes = s["c"], s["codes"]
    w = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(1)[:, : c["K"]].float()
    spread = lambda t: t.float().repeat_interleave(c["group"], dim=1)[:, : c["K"]]  # noqa: E731
    w = (w - (8.0 if s["zeros"] is None else spread(s["zeros"]))) * spread(s["scales"])
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return (torch.relu(y) if c["relu"] else y).to(s["x"].dtype)


def run(state):
    s, c = state, state["c"]
    if not own:
        return {"attend": _attend, "append": _append, "w4": _w4}[c["kind"]](s)
    lib = _lib()
    if c["kind"] == "attend":
        return lib.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"], s["scale"], window=c["window"],
                                   key_scale=s["key_scale"], value_scale=s["value_scale"], out=s["out"], workspace=s["workspace"])
    if c["kind"] == "append":
        q = lib.paged_kv_append(s["q"], s["k"], s["v"], s["keys"], s["values"], s["table"], s["pos"], sequences=s["seq"], inv_freq=s["inv_freq"],
                                interleaved=c["interleaved"], key_scale=s["key_scale"], value_scale=s["value_scale"], out=s["out"])
        return {"q": q, "keys": s["keys"], "values": s["values"]}
    return lib.matmul_w4(s["x"], s["packed"], bias=s["bias"], relu=c["relu"], out=s["out"])


# ----------------------------------------------------------------------------- floors
def work(case):
    c = case
    if c["kind"] == "w4":
        m, n, k = c["M"], c["N"], c["K"]
        groups = -(-k // c["group"])
        return {"bytes": n * k / 2 + n * groups * (2.5 if c["zeros"] else 2) + 2 * m * (n + k) + (2 * n if c["bias"] else 0), "flops": 2 * m * n * k}
    size, d = (1 if c["cache"] == "e4m3" else 2), c["dim"]
    if c["kind"] == "append":
        t = c["tokens"]
        return {"bytes": t * (d * (4 * c["heads"] + (4 + 2 * size) * c["kv_heads"]) + 12), "flops": 3 * t * c["rotary"] * (c["heads"] + c["kv_heads"])}
    keys = sum(min(n, c["window"] or n) for n in _lengths(c))
    return {"bytes": 2 * keys * c["kv_heads"] * d * size + 4 * c["sequences"] * c["heads"] * d + 4 * keys // c["page"], "flops": 4 * keys * c["heads"] * d}


# ----------------------------------------------------------------------------- in 64 bits
def _exact_attend(s):
    c, b = s["c"], s["c"]["sequences"]
    group, out = c["heads"] // c["kv_heads"], torch.zeros(b, c["heads"], c["dim"], dtype=torch.float64, device=DEV)
    ks = [1.0] * c["kv_heads"] if s["key_scale"] is None else s["key_scale"].tolist()
    vs = [1.0] * c["kv_heads"] if s["value_scale"] is None else s["value_scale"].tolist()
    table = s["table"].cpu()
    for i, n in enumerate(_lengths(c)):
        first = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n)
        page, slot = table[i][at // c["page"]].long().to(DEV), (at % c["page"]).to(DEV)
        for h in range(c["kv_heads"]):
            k, v = s["keys"][page, h, slot].double() * ks[h], s["values"][page, h, slot].double() * vs[h]
            w = torch.softmax(torch.einsum("gd,td->gt", s["q"][i, h * group:(h + 1) * group].double(), k) * s["scale"], dim=1)
            out[i, h * group:(h + 1) * group] = torch.einsum("gt,td->gd", w, v)
    return out


def _exact_append(s):
    c, r = s["c"], s["c"]["rotary"]
    first = torch.arange(0, r, 2, device=DEV) if c["interleaved"] else torch.arange(r // 2, device=DEV)
    second = first + 1 if c["interleaved"] else first + r // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(s["pos"].double(), s["inv_freq"]))[:, None]

    def turned(x):
        x = x.double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    keys, values = s["keys"].double(), s["values"].double()
    k, v = turned(s["k"]), s["v"].double()
    if s["key_scale"] is not None:
        k, v = k / s["key_scale"].double()[:, None], v / s["value_scale"].double()[:, None]
        k, v = k.clip(-448, 448), v.clip(-448, 448)
    place = s["table"].long()[s["seq"].long(), s["pos"].long().div(c["page"], rounding_mode="floor")]
    slot = s["pos"].long().remainder(c["page"])
    for h in range(c["kv_heads"]):
        keys[place, h, slot], values[place, h, slot] = k[:, h], v[:, h]
    return {"q": turned(s["q"]), "keys": keys, "values": values}


def _exact_w4(s):
    c = s["c"]
    codes = torch.empty(c["N"], 2 * s["codes"].shape[1], dtype=torch.float64, device=DEV)
    codes[:, 0::2], codes[:, 1::2] = s["codes"].remainder(16).double(), s["codes"].div(16, rounding_mode="floor").double()
    y = torch.zeros(c["M"], c["N"], dtype=torch.float64, device=DEV)
    for g in range(s["scales"].shape[1]):
        lo, hi = g * c["group"], min(c["K"], (g + 1) * c["group"])
        w = codes[:, lo:hi] - (8 if s["zeros"] is None else s["zeros"][:, g: g + 1].double())
        y += (s["x"][:, lo:hi].double() @ w.T) * s["scales"][:, g].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    return y.clip(min=0) if c["relu"] else y


def exact(case, seed):
    return {"attend": _exact_attend, "append": _exact_append, "w4": _exact_w4}[case["kind"]](_inputs(case, seed))
