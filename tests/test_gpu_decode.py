"""Decode operators on the GPU: the paged key-value cache (append with rotation, attention of one new token) and linear layers
with 4-bit weights, each against its definition in 64 bits.

Tolerances.  u(t) = eps(t) / 2 is the most a rounding to type t is off, relative to the value (bf16 2^-8, f16 2^-11, e4m3 2^-4).

attention   the result is rounded once: u |o|; the exponentials are rounded to the 16-bit type of the product with the values
            (f16 for an 8-bit cache): u_p sum p |v| / sum p at most; scores are f32 sums of at most 256 products of magnitudes up to
            about 2^6, so exponentials are off by at most 2^6 * 2^-20 = 2^-14 of themselves, the same for the sum they are divided by,
            2^-13 together
append      u |y|, and 2^-20 (|a| + |b|): cos, sin, two products and a sum in f32 are each off by 2^-22 at most; 8-bit codes below
            2^-6 have a fixed step of 2^-9, half of it is 2^-10
w4          u |y|, and 2^-14 (sum |x| |w| + |bias|): products are exact in f32, and at most 2^9 f32 additions follow one another"""
import math

import numpy as np
import pytest
import torch

from gc_b200 import lib

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "e4m3": 2.0 ** -4}
NAN_BITS = {"bf16": 0x7FFF, "f16": 0x7FFF, "e4m3": 0x7F}


def _close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    tol = tol.double().cpu() if torch.is_tensor(tol) else torch.full_like(want, tol)
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol) & ~(got == want) & ~(got.isnan() & want.isnan())
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first {i}: got {got[i]} want {want[i]} tol {tol[i]}")


def _raw(t):
    """16- or 8-bit patterns."""
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16)


def _poison(t, kind):
    _raw(t).fill_(NAN_BITS[kind])
    return t


def _cache(g, pages, kv, page, dim, kind, layout, poison=False):
    shape = (pages, kv, page, dim) if layout == "heads" else (pages, page, kv, dim)
    x = torch.randn(shape, generator=g)
    x = (x * 30 if kind == "e4m3" else x).to(T[kind]).cuda()
    if poison:
        _poison(x, kind)
    return x if layout == "heads" else x.transpose(1, 2)


def _table(g, lengths, page, spare=2):
    """A page table whose pages come in no order; entries behind a sequence's last token are no pages."""
    per = max(1, max(-(-n // page) for n in lengths)) + 1
    need = sum(-(-n // page) for n in lengths)
    order = torch.randperm(need + spare, generator=g).tolist()
    t = torch.full((len(lengths), per), -7, dtype=torch.int32)
    for s, n in enumerate(lengths):
        for e in range(-(-n // page)):
            t[s, e] = order.pop()
    return t, need + spare


def _fill(cache, table, lengths, page, g, kind):
    """Random tokens where a sequence has some; everything else keeps its bits."""
    for s, n in enumerate(lengths):
        for t in range(n):
            x = torch.randn(cache.shape[1], cache.shape[3], generator=g)
            _raw(cache)[int(table[s, t // page]), :, t % page] = _raw((x * 30 if kind == "e4m3" else x).to(T[kind]).cuda())


def _attend_want(q, keys, values, table, lengths, scale, window, page, ks, vs):
    """(out, its magnitude sum p |v|, lse) in 64 bits."""
    S, H, D = q.shape
    kv = keys.shape[1]
    G = H // kv
    out, mag, lse = torch.zeros(S, H, D, dtype=torch.float64), torch.zeros(S, H, D, dtype=torch.float64), torch.full((S, H), -math.inf, dtype=torch.float64)
    kc, vc, q = keys.double().cpu(), values.double().cpu(), q.double().cpu()
    for s, n in enumerate(lengths):
        first = max(0, n - window) if window else 0
        if n == 0:
            continue
        at = torch.arange(first, n)
        pg, sl = table[s].cpu()[at // page].long(), at % page
        k = kc[pg, :, sl].permute(1, 2, 0) * (1.0 if ks is None else ks.double().cpu()[:, None, None])    # [kv, D, T]
        v = vc[pg, :, sl].permute(1, 0, 2) * (1.0 if vs is None else vs.double().cpu()[:, None, None])    # [kv, T, D]
        x = (q[s].view(kv, G, D) @ k) * scale
        p = torch.softmax(x, dim=-1)
        out[s], mag[s], lse[s] = (p @ v).view(H, D), (p @ v.abs()).view(H, D), torch.logsumexp(x, -1).view(H)
    return out, mag, lse


def _attend_check(dtype, kind, lengths, heads, kv, dim, page, window=0, layout="heads", seed=0, qscale=1.5, **call):
    g = torch.Generator().manual_seed(seed)
    table, pages = _table(g, lengths, page)
    keys = _cache(g, pages, kv, page, dim, kind, layout, poison=True)
    values = _cache(g, pages, kv, page, dim, kind, layout, poison=True)
    _fill(keys, table, lengths, page, g, kind)
    _fill(values, table, lengths, page, g, kind)
    ks = vs = None
    if kind == "e4m3":
        ks, vs = (0.5 + torch.rand(kv, generator=g)).cuda() / 30, (0.5 + torch.rand(kv, generator=g)).cuda() / 30
    q = (torch.randn(len(lengths), heads, dim, generator=g) * qscale).to(T[dtype]).cuda()
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    lse = torch.full((len(lengths), heads), 7.0, device="cuda")
    scale = dim ** -0.5
    out = lib.paged_attention(q, keys, values, table.cuda(), lens, scale, window=window, key_scale=ks, value_scale=vs, lse=lse, **call)
    torch.cuda.synchronize()
    want, mag, wl = _attend_want(q, keys, values, table, lengths, scale, window, page, ks, vs)
    up = U["f16" if kind == "e4m3" else dtype]
    _close(out, want, U[dtype] * want.abs() + (up + 2.0 ** -13) * mag + 1e-7, f"out {lengths}")
    _close(lse, wl, 2.0 ** -13 + 2.0 ** -20 * wl.abs().nan_to_num(posinf=0.0), "lse")
    assert lib.device_error() == 0
    return out


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (8, 2), (10, 2), (7, 1), (16, 2), (16, 1), (40, 2), (33, 1)])
def test_attention_head_layouts(dtype, kind, heads, kv):
    _attend_check(dtype, kind, [1, 0, 70, 33, 257], heads, kv, 64, 16, seed=heads)


@pytest.mark.parametrize("kind", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 176, 192, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_attention_head_dims(kind, dim, layout):
    _attend_check("f16" if kind == "f16" else "bf16", kind, [17, 130, 3], 6, 2, dim, 8, layout=layout, seed=dim)


@pytest.mark.parametrize("dim", [8, 24, 72, 248])
def test_attention_dims_of_eight(dim):
    _attend_check("bf16", "bf16", [17, 130, 0, 3], 6, 2, dim, 8, seed=dim)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 64, 100, 256, 1000])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_page_sizes(page, kind):
    _attend_check("bf16", kind, [1, 63, 64, 65, 129, 300], 4, 1, 128, page, seed=page)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 65, 128, 1000])
def test_attention_windows(window):
    _attend_check("bf16", "bf16", [0, 1, 16, 64, 65, 200, 333], 8, 2, 64, 16, window=window, seed=window)


@pytest.mark.parametrize("lengths", [[0], [1], [0, 0, 0], [2], [15], [16], [17], [127], [128], [1000], [2049], [0, 2049, 0, 1, 0]], ids=str)
def test_attention_lengths(lengths):
    out = _attend_check("bf16", "bf16", lengths, 8, 8, 128, 16)
    for s, n in enumerate(lengths):
        if n == 0:
            assert not _raw(out[s]).any()      # plus zero


def test_attention_many_sequences():
    r = np.random.RandomState(5)
    _attend_check("bf16", "bf16", [int(x) for x in r.randint(0, 60, 300)], 4, 2, 64, 16)
    _attend_check("f16", "e4m3", [int(x) for x in r.randint(0, 20, 700)], 2, 1, 64, 16)


@pytest.mark.parametrize("dim,heads", [(256, 3), (176, 9), (128, 12), (64, 1)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_many_parts_to_a_unit(dim, heads, kind):
    """One KV head, a long sequence beside short ones: its softmax is cut by dozens of borders."""
    _attend_check("bf16", kind, [2500, 3, 0, 1400, 64], heads, 1, dim, 16, seed=dim)


def test_attention_more_sequences_than_a_grid_has_rows():
    """Seventy thousand sequences of one token, every seventh empty: each gives its own value row, bit for bit."""
    S, D = 70000, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    keys, values = (torch.randn(S, 1, 1, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    table = torch.randperm(S, generator=g, device="cuda").to(torch.int32)[:, None]
    lens = (torch.arange(S, device="cuda") % 7 != 0).to(torch.int32)
    q = torch.randn(S, 2, D, generator=g, device="cuda").bfloat16()
    out = lib.paged_attention(q, keys, values, table, lens, 1.0)
    want = torch.where((lens > 0)[:, None, None], values[table[:, 0].long(), :, 0], torch.zeros_like(q[:, :1])).expand(-1, 2, -1)
    assert torch.equal(out, want)
    assert lib.device_error() == 0


def test_attention_large_scores():
    """Scores in the hundreds: one token takes nearly everything, and maxima grow along the sequence."""
    # f32 scores of this size are off by up to 2^9 2^-20 instead of 2^6 2^-20: the case keeps the tolerance by having exact scores
    S, D, page = 300, 64, 16
    g = torch.Generator().manual_seed(1)
    table, pages = _table(g, [S], page)
    keys, values = _cache(g, pages, 1, page, D, "bf16", "heads"), _cache(g, pages, 1, page, D, "bf16", "heads")
    q = torch.zeros(1, 2, D)
    q[0, 0, 0], q[0, 1, 0] = 16.0, -16.0
    q = q.bfloat16().cuda()
    for t in range(S):
        keys[int(table[0, t // page]), 0, t % page, 0] = t / 8 if t % 8 == 0 else 0.5     # exact in bf16, products exact
    lens = torch.tensor([S], dtype=torch.int32).cuda()
    out = lib.paged_attention(q, keys, values, table.cuda(), lens, 1.0)
    want, mag, _ = _attend_want(q, keys, values, table, [S], 1.0, 0, page, None, None)
    _close(out, want, U["bf16"] * want.abs() + (U["bf16"] + 2.0 ** -13) * mag + 1e-7)


def test_attention_infinite_and_nan_cache_entries():
    """A NaN or an infinity among the seen values shows where the definition says so; behind the length it does not."""
    page, D, lengths = 16, 64, [40, 40, 40, 40]
    g = torch.Generator().manual_seed(2)
    table, pages = _table(g, lengths, page)
    keys, values = _cache(g, pages, 1, page, D, "bf16", "heads"), _cache(g, pages, 1, page, D, "bf16", "heads")

    def at(c, s, t):
        return c[int(table[s, t // page]), 0, t % page]
    at(keys, 0, 7)[3] = math.nan
    at(values, 1, 9)[5] = math.inf
    at(keys, 2, 41)[:] = math.nan       # behind the length, in the same page
    at(values, 2, 42)[:] = math.inf
    at(keys, 3, 11)[:] = -math.inf      # q > 0: a score of minus infinity takes no share
    q = torch.randn(4, 2, D, generator=g).abs().bfloat16().cuda()
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = lib.paged_attention(q, keys, values, table.cuda(), lens, 0.1).float().cpu()
    assert out[0].isnan().all()
    assert (out[1, :, 5] == math.inf).all() and out[1, :, :5].isfinite().all()
    want, mag, _ = _attend_want(q, keys, values, table, lengths, 0.1, 0, page, None, None)
    for s in (2, 3):
        _close(out[s], want[s], U["bf16"] * want[s].abs() + (U["bf16"] + 2.0 ** -13) * mag[s] + 1e-7)
    at(keys, 3, 11)[:] = 0
    for t in range(40):
        at(keys, 3, t)[:] = -math.inf   # every score: the softmax has no value
    out = lib.paged_attention(q, keys, values, table.cuda(), lens, 0.1)
    assert out[3].isnan().all()


def test_attention_strides_and_placement():
    """Queries and results inside larger tensors, the cache inside a joint one; what lies around them keeps its bits."""
    g = torch.Generator().manual_seed(3)
    lengths, page, kv, D, H = [100, 31, 0], 16, 2, 64, 6
    table, pages = _table(g, lengths, page)
    joint = torch.randn(pages, kv, page, 2, 3 * D, generator=g).bfloat16().cuda()
    keys, values = joint[:, :, :, 0, D:2 * D], joint[:, :, :, 1, :D]
    wide = torch.randn(3, H + 3, D + 8, generator=g).bfloat16().cuda()
    q = wide[:, 1:H + 1, :D]
    odd = torch.randn(3 * H * (D + 1) + 1, generator=g).bfloat16().cuda()
    q_odd = odd[1:].view(3, H, D + 1)[:, :, :D]             # rows on any two bytes
    q_odd.copy_(q)
    big = torch.full((3, H, D + 3), 5.0, dtype=torch.bfloat16, device="cuda")
    tab = torch.full((3, 40), 12345, dtype=torch.int32)
    tab[:, 3:3 + table.shape[1]] = table
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    want, mag, _ = _attend_want(q, keys, values, table, lengths, 0.125, 0, page, None, None)
    tol = U["bf16"] * want.abs() + (U["bf16"] + 2.0 ** -13) * mag + 1e-7
    _close(lib.paged_attention(q, keys, values, tab.cuda()[:, 3:3 + table.shape[1]], lens, 0.125), want, tol)
    lib.paged_attention(q_odd, keys, values, table.cuda(), lens, 0.125, out=big[:, :, 1:D + 1])
    _close(big[:, :, 1:D + 1], want, tol)
    assert (big[:, :, 0] == 5).all() and (big[:, :, D + 1:] == 5).all()


def test_attention_offsets_beyond_32_bits():
    """Pages more than 2^32 bytes into a cache."""
    pages, kv, page, D = 40000, 2, 256, 128     # 5.2 GB each for keys and values
    keys = torch.zeros(pages, kv, page, D, dtype=torch.bfloat16, device="cuda")
    values = torch.zeros(pages, kv, page, D, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(4)
    table = torch.tensor([[39999, 0, 35000]], dtype=torch.int32)
    for e in table[0].tolist():
        keys[e] = torch.randn(kv, page, D, generator=g).bfloat16().cuda()
        values[e] = torch.randn(kv, page, D, generator=g).bfloat16().cuda()
    q = torch.randn(1, 4, D, generator=g).bfloat16().cuda()
    lens = torch.tensor([700], dtype=torch.int32).cuda()
    out = lib.paged_attention(q, keys, values, table.cuda(), lens, 0.1)
    few = torch.tensor([[0, 1, 2]])
    want, mag, _ = _attend_want(q, keys[table[0].long()], values[table[0].long()], few, [700], 0.1, 0, page, None, None)
    _close(out, want, U["bf16"] * want.abs() + (U["bf16"] + 2.0 ** -13) * mag + 1e-7)


def test_attention_bad_pages_and_lengths_are_reported_and_not_followed():
    g = torch.Generator().manual_seed(5)
    lengths, page, D = [64, 64], 16, 64
    table, pages = _table(g, lengths, page)
    keys, values = _cache(g, pages, 2, page, D, "bf16", "heads"), _cache(g, pages, 2, page, D, "bf16", "heads")
    q = torch.randn(2, 4, D, generator=g).bfloat16().cuda()
    lens = torch.tensor(lengths, dtype=torch.int32).cuda()
    good = lib.paged_attention(q, keys, values, table.cuda(), lens, 0.125)
    assert lib.device_error() == 0
    bad = table.clone()
    bad[0, 1], bad[0, 2] = 1 << 30, -3
    out = lib.paged_attention(q, keys, values, bad.cuda(), lens, 0.125)
    assert lib.device_error() == 9 and lib.device_error() == 0
    assert torch.equal(out[1], good[1])                     # the other sequence is untouched by it
    k2, v2 = torch.cat([keys, torch.zeros_like(keys[:1])]), torch.cat([values, torch.zeros_like(values[:1])])
    bad[0, 1] = bad[0, 2] = pages                           # tokens of unknown pages count as zeros
    assert torch.equal(lib.paged_attention(q, k2, v2, bad.cuda(), lens, 0.125), out)
    short = table[:, :4].contiguous()
    cut = lib.paged_attention(q, keys, values, short.cuda(), torch.tensor([64, 1 << 30], dtype=torch.int32).cuda(), 0.125)
    assert lib.device_error() == 9
    assert torch.equal(cut, good)


def test_attention_same_bits_every_time_and_on_other_streams():
    g = torch.Generator().manual_seed(6)
    lengths, page, D = [3000, 10, 777, 0, 1500], 16, 128
    table, pages = _table(g, lengths, page)
    keys, values = _cache(g, pages, 2, page, D, "bf16", "heads"), _cache(g, pages, 2, page, D, "bf16", "heads")
    q = torch.randn(5, 8, D, generator=g).bfloat16().cuda()
    lens, tab = torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda()
    first = lib.paged_attention(q, keys, values, tab, lens, 0.1)
    for _ in range(5):
        assert torch.equal(lib.paged_attention(q, keys, values, tab, lens, 0.1), first)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):                                     # calls that overlap, each with a workspace of its own
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(lib.paged_attention(q, keys, values, tab, lens, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)


def test_attention_and_append_in_captured_graphs():
    """A captured step follows its lengths and positions in device memory; two graphs replayed in turn do not disturb each other."""
    g = torch.Generator().manual_seed(7)
    page, D, kv, H, S = 16, 64, 2, 8, 3
    room = 400
    table, pages = _table(g, [room] * S, page)
    tab = table.cuda()
    inv = (1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).cuda()

    def state(seed):
        gg = torch.Generator().manual_seed(seed)
        return {"keys": _cache(gg, pages, kv, page, D, "bf16", "heads"), "values": _cache(gg, pages, kv, page, D, "bf16", "heads"),
                "q": torch.randn(S, H, D, generator=gg).bfloat16().cuda(), "k": torch.randn(S, kv, D, generator=gg).bfloat16().cuda(),
                "v": torch.randn(S, kv, D, generator=gg).bfloat16().cuda(), "lens": torch.tensor([5, 60, 200], dtype=torch.int32).cuda()}

    def step(st):
        q = lib.paged_kv_append(st["q"], st["k"], st["v"], st["keys"], st["values"], tab, st["lens"] - 1, inv_freq=inv)
        return lib.paged_attention(q, st["keys"], st["values"], tab, st["lens"], 0.125)

    states = [state(1), state(2)]
    step(states[0])
    torch.cuda.synchronize()
    graphs = []
    for st in states:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            st["out"] = step(st)
        graphs.append(gr)
    for n in ([5, 60, 200], [1, 399, 17], [0, 2, 400]):
        for st, gr in zip(states, graphs):
            st["lens"].copy_(torch.tensor(n, dtype=torch.int32))
            gr.replay()
        torch.cuda.synchronize()
        got = [st["out"].clone() for st in states]
        for st, o in zip(states, got):
            assert torch.equal(step(st), o)
    assert lib.device_error() == 0


def test_attention_keys_and_values_laid_out_differently():
    """Keys with heads outside tokens, values with tokens outside heads, and another distance between pages."""
    g = torch.Generator().manual_seed(12)
    lengths, kv, D, H = [200, 0, 33, 1], 2, 128, 8
    for page in (16, 24):
        table, pages = _table(g, lengths, page)
        for kk, kind in (("bf16", "bf16"), ("bf16", "e4m3")):
            keys = _cache(g, pages, kv, page, D, kind, "heads")
            values = _cache(g, 2 * pages, kv, page, D, kind, "tokens")[::2]
            ks = vs = torch.full((kv,), 0.03, device="cuda") if kind == "e4m3" else None
            q = torch.randn(4, H, D, generator=g).bfloat16().cuda()
            lens = torch.tensor(lengths, dtype=torch.int32).cuda()
            out = lib.paged_attention(q, keys, values, table.cuda(), lens, 0.08, key_scale=ks, value_scale=vs)
            want, mag, _ = _attend_want(q, keys, values, table, lengths, 0.08, 0, page, ks, vs)
            _close(out, want, U["bf16"] * want.abs() + (U["f16" if kind == "e4m3" else "bf16"] + 2.0 ** -13) * mag + 1e-7)


def test_attention_negative_lengths_and_scales():
    g = torch.Generator().manual_seed(13)
    lengths, page, D = [90, 17], 16, 64
    table, pages = _table(g, lengths, page)
    for kind in ("bf16", "e4m3"):
        keys, values = _cache(g, pages, 1, page, D, kind, "heads"), _cache(g, pages, 1, page, D, kind, "heads")
        ks = vs = torch.full((1,), 0.03, device="cuda") if kind == "e4m3" else None
        q = torch.randn(2, 3, D, generator=g).bfloat16().cuda()
        lse = torch.zeros(2, 3, device="cuda")
        out = lib.paged_attention(q, keys, values, table.cuda(), torch.tensor([90, -5], dtype=torch.int32).cuda(), -0.2, key_scale=ks, value_scale=vs, lse=lse)
        want, mag, wl = _attend_want(q, keys, values, table, [90, 0], -0.2, 0, page, ks, vs)
        _close(out, want, U["bf16"] * want.abs() + (U["f16" if kind == "e4m3" else "bf16"] + 2.0 ** -13) * mag + 1e-7)
        assert (lse[1] == -math.inf).all() and not _raw(out[1]).any()
        flat = lib.paged_attention(q, keys, values, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), 0.0, key_scale=ks, value_scale=vs)
        want, mag, _ = _attend_want(q, keys, values, table, lengths, 0.0, 0, page, ks, vs)      # the mean of the values
        _close(flat, want, U["bf16"] * want.abs() + (U["f16" if kind == "e4m3" else "bf16"] + 2.0 ** -13) * mag + 1e-7)


@pytest.mark.parametrize("kind", ["f16", "e4m3"])
def test_attention_one_large_share_and_a_long_tail(kind):
    """One token takes half of the softmax, thousands of others below 2^-12 of it the other half: none of them may vanish.  Their
    exponentials are far below f16's smallest normal number."""
    S, D, page = 20000, 64, 32
    table = torch.arange(S // page, dtype=torch.int32)[None].cuda()
    keys = torch.zeros(S // page, 1, page, D).to(T[kind]).cuda()
    values = torch.ones(S // page, 1, page, D).to(T[kind]).cuda()
    keys[3, 0, 5, 0] = 1.0
    values[3, 0, 5] = -1.0
    q = torch.zeros(1, 1, D, dtype=torch.float16)
    q[0, 0, 0] = 10.0
    q = q.cuda()
    one = torch.ones(1, device="cuda") if kind == "e4m3" else None
    out = lib.paged_attention(q, keys, values, table, torch.tensor([S], dtype=torch.int32).cuda(), 1.0, key_scale=one, value_scale=one)
    w = math.exp(10.0)
    want = torch.full((1, 1, D), (S - 1 - w) / (S - 1 + w), dtype=torch.float64)
    _close(out, want, U["f16"] * want.abs() + (U["f16"] + 2.0 ** -13))
    q[0, 0, 0] = 18.0           # the others: e^-18, below 2^-25
    keys[3, 0, 5, 0] = 1.0
    out = lib.paged_attention(q, keys, values, table, torch.tensor([S], dtype=torch.int32).cuda(), 1.0, key_scale=one, value_scale=one)
    w = math.exp(18.0)
    want = torch.full((1, 1, D), (S - 1 - w) / (S - 1 + w), dtype=torch.float64)
    _close(out, want, U["f16"] * want.abs() + (U["f16"] + 2.0 ** -13))


def test_first_use_of_a_variant_inside_a_capture():
    """A kernel variant that no call has used yet, captured and replayed."""
    g = torch.Generator().manual_seed(14)
    lengths, page, D = [300, 77], 16, 96
    table, pages = _table(g, lengths, page)
    keys, values = _cache(g, pages, 1, page, D, "f16", "heads"), _cache(g, pages, 1, page, D, "f16", "heads")
    q = torch.randn(2, 13, D, generator=g).half().cuda()
    lens, tab = torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda()
    codes, scales = torch.randint(0, 256, (48, 300), generator=g, dtype=torch.uint8).cuda(), torch.rand(48, 10, generator=g).half().cuda()
    w = lib.pack_w4(codes, scales, 600, 64, zeros=torch.randint(0, 16, (48, 10), generator=g, dtype=torch.uint8).cuda())
    x = torch.randn(11, 600, generator=g).half().cuda()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = lib.paged_attention(q, keys, values, tab, lens, 0.1)
        y = lib.matmul_w4(x, w)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, lib.paged_attention(q, keys, values, tab, lens, 0.1)) and torch.equal(y, lib.matmul_w4(x, w))
    want, mag, _ = _attend_want(q, keys, values, table, lengths, 0.1, 0, page, None, None)
    _close(out, want, U["f16"] * want.abs() + (U["f16"] + 2.0 ** -13) * mag + 1e-7)


# ----------------------------------------------------------------------------- append
def _rotated(x, pos, inv, interleaved):
    """(rotated, |a| + |b| of each element's pair) in 64 bits."""
    x = x.double().cpu()
    if inv is None:
        return x, torch.zeros_like(x)
    ang = pos.double().cpu()[:, None, None] * inv.cpu()
    c, s = torch.cos(ang), torch.sin(ang)
    n = inv.numel()
    i0 = torch.arange(n) * 2 if interleaved else torch.arange(n)
    i1 = i0 + (1 if interleaved else n)
    y, m = x.clone(), torch.zeros_like(x)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    m[..., i0] = m[..., i1] = a.abs() + b.abs()
    return y, m


def _append_check(dtype, kind, tokens, heads, kv, dim, rotary, interleaved, page, layout="heads", seq=None, pos=None, in_place=False, odd=False, seed=0, with_q=True):
    g = torch.Generator().manual_seed(seed)
    if seq is None:
        seq, pos = list(range(tokens)), [int(x) for x in torch.randint(0, 5 * page, (tokens,), generator=g)]
    sequences = max(max(seq), 0) + 1
    lengths = [max([p + 1 for s2, p in zip(seq, pos) if s2 == s] + [0]) for s in range(sequences)]
    per = max(-(-n // page) for n in lengths) + 1
    touched = sorted({(s, p // page) for s, p in zip(seq, pos) if s >= 0 and p >= 0})
    pages = len(touched) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((sequences, per), -1, dtype=torch.int32)
    for i, (s, e) in enumerate(touched):
        table[s, e] = order[i]
    keys, values = _cache(g, pages, kv, page, dim, kind, layout), _cache(g, pages, kv, page, dim, kind, layout)
    before = _raw(keys).clone(), _raw(values).clone()
    ks = vs = None
    if kind == "e4m3":
        ks, vs = (0.5 + torch.rand(kv, generator=g)).cuda() / 30, (0.5 + torch.rand(kv, generator=g)).cuda() / 30
    width = (heads + 2 * kv) * dim + (3 if odd else 0)
    qkv = torch.randn(tokens, width, generator=g).to(T[dtype]).cuda()
    parts = [(0, heads), (heads, kv), (heads + kv, kv)]
    q, k, v = (qkv[:, a * dim:(a + n) * dim].unflatten(1, (n, dim)) for a, n in parts)
    inv = None if not rotary else (1.0 / 10000.0 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).cuda()
    P, Q = torch.tensor(pos, dtype=torch.int32), torch.tensor(seq, dtype=torch.int32)
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    out = lib.paged_kv_append(q if with_q else None, k, v, keys, values, table.cuda(), P.cuda(), sequences=Q.cuda(), inv_freq=inv, interleaved=interleaved,
                              key_scale=ks, value_scale=vs, out=q if in_place else torch.full_like(q0, 9.0) if with_q else None)
    torch.cuda.synchronize()
    assert lib.device_error() == 0
    live = [i for i in range(tokens) if seq[i] >= 0 and pos[i] >= 0]
    dead = [i for i in range(tokens) if i not in set(live)]
    if with_q:
        want, pair = _rotated(q0, P, inv, interleaved)
        _close(out[live], want[live], U[dtype] * want[live].abs() + 2.0 ** -20 * pair[live], "q")
        assert torch.equal(out[dead], q0[dead] if in_place else torch.full_like(q0[dead], 9.0))
    else:
        assert out is None
    assert torch.equal(k, k0) and torch.equal(v, v0)
    pg = torch.tensor([int(table[seq[i], pos[i] // page]) for i in live], dtype=torch.long)
    sl = torch.tensor([pos[i] % page for i in live], dtype=torch.long)
    for cache, x, scale, old, rot in ((keys, k0, ks, before[0], inv), (values, v0, vs, before[1], None)):
        want, pair = _rotated(x, P, rot, interleaved)
        tol = 2.0 ** -20 * pair
        if scale is not None:
            sc = scale.double().cpu()[:, None]
            want, tol = (want / sc).clamp(-448, 448), tol / sc + 2.0 ** -10
        got = cache[pg.cuda(), :, sl.cuda()]
        _close(got, want[live], U[kind] * want[live].abs() + tol[live], "cache")
        if rot is None and scale is None:
            assert torch.equal(_raw(got), _raw(x[live]))       # values are copied bit for bit
        _raw(cache)[pg.cuda(), :, sl.cuda()] = old[pg.cuda(), :, sl.cuda()]
        assert torch.equal(_raw(cache), old)                   # nothing else has changed


@pytest.mark.parametrize("dtype,kind", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("heads,kv,dim,rotary,interleaved", [(8, 2, 128, 128, False), (8, 2, 128, 128, True), (4, 4, 64, 32, False), (4, 4, 64, 32, True),
                                                             (7, 1, 80, 40, False), (7, 1, 80, 40, True), (5, 5, 96, 96, False), (2, 1, 256, 64, False),
                                                             (3, 1, 16, 6, False), (3, 1, 16, 6, True), (3, 3, 48, 4, True), (6, 2, 112, 0, False), (16, 1, 176, 176, True)])
def test_append_shapes(dtype, kind, heads, kv, dim, rotary, interleaved):
    _append_check(dtype, kind, 9, heads, kv, dim, rotary, interleaved, 16, seed=dim + rotary)


@pytest.mark.parametrize("dim,rotary,interleaved", [(8, 8, False), (24, 2, False), (72, 72, False), (72, 18, True), (248, 248, False)])
def test_append_dims_of_eight(dim, rotary, interleaved):
    _append_check("bf16", "bf16", 5, 3, 1, dim, rotary, interleaved, 16)


@pytest.mark.parametrize("page", [1, 3, 24, 128])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_append_pages_and_layouts(page, layout, kind):
    seq = [0] * 40 + [2] * 7 + [1]
    pos = list(range(3, 43)) + list(range(7)) + [100]
    _append_check("bf16", kind, 48, 8, 2, 64, 64, False, page, layout, seq, pos)


def test_append_padding_leaves_rows_as_they_were():
    seq, pos = [0, -1, 1, 2, -1, 3], [5, 7, -1, 0, -1, 9]
    for in_place in (False, True):
        _append_check("bf16", "bf16", 6, 4, 2, 64, 64, False, 16, seq=seq, pos=pos, in_place=in_place)


def test_append_in_place_unaligned_and_without_queries():
    for inter in (False, True):
        _append_check("bf16", "bf16", 33, 8, 2, 128, 128, inter, 16, in_place=True)
        _append_check("f16", "e4m3", 5, 8, 2, 128, 64, inter, 16, odd=True, in_place=True)
        _append_check("bf16", "bf16", 1, 1, 1, 64, 64, inter, 16, odd=True)
    _append_check("bf16", "bf16", 12, 4, 2, 64, 64, False, 16, with_q=False)


def test_append_far_positions():
    """Angles of positions up to 2^30 keep their fraction: the table has one entry for each page, most of them no page."""
    page = 1 << 20
    g = torch.Generator().manual_seed(0)
    pos = torch.tensor([0, 1, 999999, (1 << 24) + 1, (1 << 30) - 1], dtype=torch.int32)
    table = torch.full((5, 1024), -1, dtype=torch.int32)
    for i, p in enumerate(pos.tolist()):
        table[i, p // page] = i
    q = torch.randn(5, 2, 64, generator=g).bfloat16().cuda()
    k = torch.randn(5, 1, 64, generator=g).bfloat16().cuda()
    cache = torch.zeros(5, 1, page, 64, dtype=torch.bfloat16, device="cuda")
    inv = (1.0 / 10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)).cuda()
    out = lib.paged_kv_append(q, k, k, cache, torch.zeros_like(cache), table.cuda(), pos.cuda(), inv_freq=inv)
    want, pair = _rotated(q, pos, inv, False)
    _close(out, want, U["bf16"] * want.abs() + 2.0 ** -20 * pair)
    want, pair = _rotated(k, pos, inv, False)
    _close(cache[torch.arange(5).cuda(), 0, (pos % page).long().cuda()], want[:, 0], U["bf16"] * want[:, 0].abs() + 2.0 ** -20 * pair[:, 0])


def test_append_special_values():
    """Infinities and NaN: limited to +-448 in 8 bits, NaN stays NaN."""
    page, D = 16, 16
    k = torch.zeros(1, 1, D)
    k[0, 0, :6] = torch.tensor([math.inf, -math.inf, math.nan, 1e5, 0.0, -0.0])
    table = torch.zeros(1, 1, dtype=torch.int32).cuda()
    pos = torch.tensor([3], dtype=torch.int32).cuda()
    for kind in ("bf16", "e4m3"):
        keys = torch.zeros(1, 1, page, D).to(T[kind]).cuda()
        values = torch.zeros_like(keys)
        x = k.bfloat16().cuda()
        lib.paged_kv_append(None, x, x, keys, values, table, pos)
        got = values[0, 0, 3].float().cpu()
        if kind == "bf16":
            assert torch.equal(_raw(values[0, 0, 3]), _raw(x[0, 0]))
        else:
            assert got[:2].tolist() == [448.0, -448.0] and got[2].isnan() and got[3] == 448.0 and got[4] == 0


def test_append_bad_pages_are_reported_and_not_written():
    g = torch.Generator().manual_seed(1)
    page, D = 16, 64
    keys, values = _cache(g, 4, 2, page, D, "bf16", "heads"), _cache(g, 4, 2, page, D, "bf16", "heads")
    k0, v0 = keys.clone(), values.clone()
    table = torch.tensor([[1, 4], [-1, 2], [3, 1 << 30]], dtype=torch.int32).cuda()
    q = torch.randn(4, 4, D, generator=g).bfloat16().cuda()
    k = torch.randn(4, 2, D, generator=g).bfloat16().cuda()
    inv = (1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).cuda()
    pos = torch.tensor([16, 0, 32, 5], dtype=torch.int32)             # page 4 of 4, page -1, beyond the table, no such sequence
    out = lib.paged_kv_append(q, k, k, keys, values, table, pos.cuda(), sequences=torch.tensor([0, 1, 2, 3], dtype=torch.int32).cuda(), inv_freq=inv)
    assert lib.device_error() == 9 and lib.device_error() == 0
    assert torch.equal(keys, k0) and torch.equal(values, v0)
    want, pair = _rotated(q, pos, inv, False)
    _close(out, want, U["bf16"] * want.abs() + 2.0 ** -20 * pair)      # the queries are turned all the same


# ----------------------------------------------------------------------------- 4-bit weights
def _w4_check(M, N, K, group, zeros, bias, relu, dtype, seed=0, xstride=0, ystride=0, xoff=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, dtype=torch.uint8)
    scales = (0.5 + torch.rand(N, groups, generator=g)).to(T[dtype])
    zs = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    x = torch.randn(M, K, generator=g).to(T[dtype])
    b = torch.randn(N, generator=g).to(T[dtype]) if bias else None
    w = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :K].double()
    spread = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    w = (w - (8 if zs is None else spread(zs))) * spread(scales)
    want = x.double() @ w.T + (b.double() if bias else 0)
    mag = x.double().abs() @ w.abs().T + (b.double().abs() if bias else 0)
    want = want.clamp(min=0) if relu else want
    packed = lib.pack_w4(codes.cuda(), scales.cuda(), K, group, zeros=None if zs is None else zs.cuda())
    xs = torch.full((M * (K + xstride) + xoff,), math.nan, dtype=T[dtype], device="cuda")[xoff:].view(M, K + xstride)[:, :K]
    xs.copy_(x)
    whole = torch.full((M, N + ystride), 3.0, dtype=T[dtype], device="cuda")
    got = lib.matmul_w4(xs, packed, bias=None if b is None else b.cuda(), relu=relu, out=whole[:, :N] if ystride else None)
    torch.cuda.synchronize()
    _close(got, want, U[dtype] * want.abs() + 2.0 ** -14 * mag, f"{M}x{N}x{K}")
    assert (whole[:, N:] == 3).all()
    assert lib.device_error() == 0
    return packed


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16])
def test_w4_groups(dtype, group, zeros, M):
    _w4_check(M, 160, 640, group, zeros, M % 2 == 1, M == 8, dtype, seed=M + group)


@pytest.mark.parametrize("M,N,K,group", [(1, 1, 1, 32), (1, 1, 2, 128), (2, 17, 33, 32), (5, 15, 127, 64), (16, 129, 129, 128), (7, 1001, 513, 32), (1, 64, 4096, 4096),
                                         (4, 2048, 1000, 1024), (17, 100, 200, 64), (40, 333, 384, 128), (65, 48, 1030, 256), (1, 5000, 64, 64), (13, 31, 8191, 128)])
@pytest.mark.parametrize("zeros", [False, True])
def test_w4_odd_sizes(M, N, K, group, zeros):
    _w4_check(M, N, K, group, zeros, True, False, "bf16", seed=K)
    _w4_check(M, N, K, group, zeros, False, True, "f16", seed=N)


def test_w4_layers_of_the_decoder_block():
    for M, N, K in [(1, 4096, 4096), (16, 11008, 4096), (8, 4096, 11008), (2, 28672, 1024)]:
        _w4_check(M, N, K, 128, False, False, False, "bf16", seed=M)


def test_w4_strides():
    for xs, ys, off in [(8, 8, 0), (1, 1, 0), (0, 0, 1), (3, 5, 1), (4, 0, 4)]:
        _w4_check(6, 200, 384, 128, True, True, False, "bf16", xstride=xs, ystride=ys, xoff=off)
        _w4_check(1, 72, 520, 32, False, False, False, "f16", xstride=xs, ystride=ys, xoff=off)


def test_w4_special_values_stay_in_their_rows():
    """An infinity or a NaN in one row of x does not reach the other rows; one beyond K is not read."""
    g = torch.Generator().manual_seed(0)
    codes, scales = torch.randint(0, 256, (96, 100), generator=g, dtype=torch.uint8).cuda(), torch.rand(96, 2, generator=g).bfloat16().cuda()
    p = lib.pack_w4(codes, scales, 200, 128)
    x = torch.randn(4, 200, generator=g).bfloat16().cuda()
    clean = lib.matmul_w4(x, p)
    x[1, 7], x[2, 199] = math.nan, math.inf
    y = lib.matmul_w4(x, p)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    assert y[1].isnan().all() and not y[2].isfinite().any()
    assert torch.equal(lib.matmul_w4(x, p, relu=True)[1].isnan(), y[1].isnan())


def test_w4_same_bits_every_time_and_rows_alone():
    """A row's result does not depend on the call before it or, within sixteen rows, on a second call."""
    g = torch.Generator().manual_seed(0)
    codes, scales = torch.randint(0, 256, (4096, 1024), generator=g, dtype=torch.uint8).cuda(), torch.rand(4096, 16, generator=g).bfloat16().cuda()
    p = lib.pack_w4(codes, scales, 2048, 128)
    x = torch.randn(16, 2048, generator=g).bfloat16().cuda()
    y = lib.matmul_w4(x, p)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        assert torch.equal(lib.matmul_w4(x, p), y)
        with torch.cuda.stream(other):
            z = lib.matmul_w4(x, p)
        other.synchronize()
        assert torch.equal(z, y)


def test_w4_long_rows_and_what_does_not_fit():
    """Rows of x that only a cluster's shared memory holds, fewer rows at a time where sixteen do not fit, and too long ones."""
    _w4_check(1, 40, 60000, 128, False, False, False, "bf16")
    _w4_check(16, 24, 30001, 64, True, True, False, "f16")
    _w4_check(3, 33, 100000, 256, False, False, False, "bf16")
    codes, scales = torch.zeros(16, 130000, dtype=torch.uint8, device="cuda"), torch.ones(16, 1, dtype=torch.bfloat16, device="cuda")
    p = lib.pack_w4(codes, scales, 260000, 260096)
    with pytest.raises(lib.GcB200Error, match="does not fit"):
        lib.matmul_w4(torch.zeros(1, 260000, dtype=torch.bfloat16, device="cuda"), p)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_w4_rows_of_unequal_magnitude(dtype):
    """Rows, and the k blocks of a row, whose magnitudes lie far apart, subnormal ones and zeros among them."""
    g = torch.Generator().manual_seed(3)
    M, N, K = 12, 64, 768
    codes, scales = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8), (0.5 + torch.rand(N, K // 128, generator=g)).to(T[dtype])
    w = (torch.stack([codes & 15, codes >> 4], -1).flatten(1).double() - 8) * scales.double().repeat_interleave(128, 1)
    e = torch.randint(-30, 31, (M, K // 128), generator=g) if dtype == "bf16" else torch.randint(-9, 9, (M, K // 128), generator=g)
    x = torch.randn(M, K, generator=g) * (2.0 ** e).repeat_interleave(128, 1)
    x[0] = 0
    x[1] = 1e-40 if dtype == "bf16" else 6e-8
    x[2, :128] = 3e38 if dtype == "bf16" else 6e4
    x[2, 128:] = 0
    x = x.to(T[dtype])
    y = lib.matmul_w4(x.cuda(), lib.pack_w4(codes.cuda(), scales.cuda(), K, 128))
    want, mag = x.double() @ w.T, x.double().abs() @ w.abs().T
    top = 3.39e38 if dtype == "bf16" else 65504.0
    ok = mag < top / 2          # what is larger may overflow the result's type, or the f32 sum
    _close(y.cpu().double()[ok], want[ok], (U[dtype] * want.abs() + 2.0 ** -14 * mag + torch.finfo(T[dtype]).smallest_normal * U[dtype] * 2)[ok])


# ----------------------------------------------------------------------------- refusals, and the operators as a run
def test_python_refusals():
    cache = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    good = dict(q=q, key_cache=cache, value_cache=cache, page_table=table, lengths=lens, scale=1.0)
    lib.paged_attention(**good)
    f8 = cache.to(torch.float8_e4m3fn)
    for bad in [dict(q=q.float()), dict(q=q.half()), dict(q=q.cpu()), dict(q=q[0]), dict(q=q[:1]), dict(key_cache=cache.cpu()), dict(key_cache=cache[0]),
                dict(value_cache=f8), dict(value_cache=cache[:2]), dict(page_table=table.long()), dict(page_table=table.cpu()), dict(lengths=lens.long()),
                dict(lengths=lens[:1]), dict(lengths=None), dict(lengths=torch.ones(4, dtype=torch.int32, device="cuda")[::2]), dict(out=q.float()), dict(out=q[:, :2]),
                dict(lse=torch.zeros(2, 4, dtype=torch.float64, device="cuda")), dict(lse=torch.zeros(4, 2, device="cuda")),
                dict(key_scale=torch.ones(1, device="cuda")), dict(key_scale=torch.ones(2, device="cuda", dtype=torch.float64)),
                dict(workspace=torch.zeros(64, device="cuda")), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))]:
        with pytest.raises(AssertionError):
            lib.paged_attention(**{**good, **bad})
    for bad in [dict(key_scale=torch.ones(2, device="cuda")), dict(q=q[:, :3]), dict(window=-1),
                dict(key_cache=torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16, device="cuda")[..., :64], value_cache=torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16, device="cuda")[..., :64])]:
        with pytest.raises(lib.GcB200Error):
            lib.paged_attention(**{**good, **bad})
    good = dict(q=q, k=k, v=k, key_cache=cache, value_cache=cache, page_table=table, positions=lens)
    inv = torch.ones(32, dtype=torch.float64, device="cuda")
    lib.paged_kv_append(**good, inv_freq=inv)
    for bad in [dict(q=q.half()), dict(k=k.cpu()), dict(v=k[:1]), dict(v=k[:, :1]), dict(positions=lens.long()), dict(positions=None), dict(sequences=lens[:1]),
                dict(inv_freq=inv.float()), dict(inv_freq=inv.cpu()), dict(out=q[:, :2]), dict(key_cache=cache.half())]:
        with pytest.raises(AssertionError):
            lib.paged_kv_append(**{**good, **bad})
    with pytest.raises(lib.GcB200Error):
        lib.paged_kv_append(**good, inv_freq=torch.ones(33, dtype=torch.float64, device="cuda"))
    codes, scales = torch.zeros(32, 64, dtype=torch.uint8, device="cuda"), torch.ones(32, 1, dtype=torch.bfloat16, device="cuda")
    p = lib.pack_w4(codes, scales, 128, 128)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device="cuda")
    lib.matmul_w4(x, p)
    for f in [lambda: lib.matmul_w4(x.half(), p), lambda: lib.matmul_w4(x[:, :64], p), lambda: lib.matmul_w4(x.cpu(), p, out=x), lambda: lib.matmul_w4(x, p, out=x),
              lambda: lib.matmul_w4(x, p, bias=scales.view(-1).float()), lambda: lib.matmul_w4(x, p, bias=scales.view(-1)[:31]),
              lambda: lib.matmul_w4(x, lib.W4Weights(p.packed[:-16], 32, 128, 128, False, torch.bfloat16)), lambda: lib.pack_w4(codes.cpu(), scales, 128, 128),
              lambda: lib.pack_w4(codes, scales.float(), 128, 128), lambda: lib.pack_w4(codes, scales, 130, 128), lambda: lib.pack_w4(codes, scales, 128, 64)]:
        with pytest.raises(AssertionError):
            f()
    with pytest.raises(lib.GcB200Error):
        lib.pack_w4(codes, scales, 128, 48)
    assert lib.matmul_w4(x[:0], p).shape == (0, 32)
    assert lib.device_error() == 0


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_block_step_by_step(kind):
    """A prompt, then single tokens through the attention half of a decoder block: 4-bit projections, append, attention, 4-bit
    projection.  Each step's intermediate tensors are checked where they are produced; the run is that of a program."""
    g = torch.Generator().manual_seed(11)
    hidden, H, kv, D, page, S = 256, 8, 2, 64, 16, 3
    width = (H + 2 * kv) * D

    def layer(n, k, seed):
        gg = torch.Generator().manual_seed(seed)
        codes = torch.randint(0, 256, (n, k // 2), generator=gg, dtype=torch.uint8)
        scales = ((0.5 + torch.rand(n, k // 128, generator=gg)) * 0.2 * k ** -0.5).bfloat16()
        w = (torch.stack([codes & 15, codes >> 4], -1).flatten(1).double() - 8) * scales.double().repeat_interleave(128, 1)
        return lib.pack_w4(codes.cuda(), scales.cuda(), k, 128), w

    wqkv, wqkv64 = layer(width, hidden, 1)
    wo, wo64 = layer(hidden, H * D, 2)
    table, pages = _table(g, [100] * S, page)
    tab = table.cuda()
    keys, values = _cache(g, pages, kv, page, D, kind, "heads", poison=True), _cache(g, pages, kv, page, D, kind, "heads", poison=True)
    ks = vs = torch.full((kv,), 0.02, device="cuda") if kind == "e4m3" else None
    inv = (1.0 / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)).cuda()
    lens = torch.zeros(S, dtype=torch.int32)

    def project(x):
        qkv = lib.matmul_w4(x, wqkv)
        q, k, v = qkv.split([H * D, kv * D, kv * D], dim=1)
        return q.unflatten(1, (H, D)), k.unflatten(1, (kv, D)), v.unflatten(1, (kv, D))

    # prompts of 5, 1 and 30 tokens in one call, padded to 40 rows
    n = [5, 1, 30]
    seq = torch.tensor([s for s in range(S) for _ in range(n[s])] + [-1] * 4, dtype=torch.int32)
    pos = torch.tensor([p for s in range(S) for p in range(n[s])] + [-1] * 4, dtype=torch.int32)
    x = torch.randn(40, hidden, generator=g).bfloat16().cuda()
    q, k, v = project(x)
    lib.paged_kv_append(q, k, v, keys, values, tab, pos.cuda(), sequences=seq.cuda(), inv_freq=inv, key_scale=ks, value_scale=vs)
    lens += torch.tensor(n, dtype=torch.int32)
    for step in range(6):
        lens += 1
        dl = lens.cuda()
        x = torch.randn(S, hidden, generator=g).bfloat16().cuda()
        q, k, v = project(x)
        want = x.double().cpu() @ wqkv64.T
        _close(q.flatten(1), want[:, :H * D], U["bf16"] * want[:, :H * D].abs() + 2.0 ** -14 * (x.double().cpu().abs() @ wqkv64.abs().T)[:, :H * D])
        rq = lib.paged_kv_append(q, k, v, keys, values, tab, dl - 1, inv_freq=inv, key_scale=ks, value_scale=vs)
        o = lib.paged_attention(rq, keys, values, tab, dl, D ** -0.5, key_scale=ks, value_scale=vs)
        want, mag, _ = _attend_want(rq, keys, values, table, lens.tolist(), D ** -0.5, 0, page, ks, vs)
        up = U["f16" if kind == "e4m3" else "bf16"]
        _close(o, want, U["bf16"] * want.abs() + (up + 2.0 ** -13) * mag + 1e-7, f"step {step}")
        y = lib.matmul_w4(o.flatten(1), wo, relu=True)
        o64 = o.double().cpu().flatten(1)
        want = (o64 @ wo64.T).clamp(min=0)
        _close(y, want, U["bf16"] * want.abs() + 2.0 ** -14 * (o64.abs() @ wo64.abs().T))
    assert lib.device_error() == 0
