"""Decode operators without a device: what the entry points refuse, and the index arithmetic that decides which memory the
kernels of the paged cache touch (compiled here for the host)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from gc_b200 import lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, NO_DEVICE = 0, 1, 3
BF16, F16, E4M3 = 2, 1, 10
P = 1 << 20   # an address that is aligned and never followed


def _i64s(*v):
    return (C.c_int64 * len(v))(*v)


def _desc(**kw):
    d = lib.PagedCacheDesc()
    base = dict(dtype=BF16, cache_dtype=BF16, pages=8, page_size=16, kv_heads=2, head_dim=64, keys=P, values=P, page_table=P, sequences=3,
                max_pages=4, page_table_stride=4)
    base.update({k: v for k, v in kw.items() if k not in ("key_stride", "value_stride")})
    for k, v in base.items():
        setattr(d, k, v)
    dense = (d.kv_heads * d.page_size * d.head_dim, d.page_size * d.head_dim, d.head_dim)
    d.key_stride = (C.c_int64 * 3)(*kw.get("key_stride", dense))
    d.value_stride = (C.c_int64 * 3)(*kw.get("value_stride", dense))
    return d


BAD_CACHES = [
    dict(dtype=3), dict(cache_dtype=F16), dict(dtype=F16, cache_dtype=BF16), dict(keys=None), dict(values=None), dict(page_table=None),
    dict(pages=0), dict(page_size=0), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=4), dict(head_dim=68), dict(head_dim=264),
    dict(cache_dtype=E4M3, head_dim=72), dict(key_scale=P), dict(value_scale=P), dict(keys=P + 8), dict(values=P + 2),
    dict(key_stride=(2048, 1024, 60)), dict(value_stride=(2044, 1024, 64)), dict(key_stride=(2048, -1024, 64)), dict(page_table_stride=3),
    dict(max_pages=1 << 28, page_table_stride=1 << 28), dict(sequences=-1), dict(max_pages=-1),
]


def _append(d, heads=4, tokens=3, q=P, k=P, v=P, out=P, seq=None, pos=P, inv=None, rotary=0):
    s = _i64s(heads * 64, 64)
    return lib.load().gcb200_paged_kv_append(C.byref(d) if d is not None else None, q, s, heads, k, s, v, s, out, s, seq, pos, tokens, inv, rotary, 0, None)


def _attend(d, heads=4, q=P, out=P, lengths=P, window=0, ws=P, ws_bytes=1 << 30):
    s = _i64s(heads * 64, 64)
    return lib.load().gcb200_paged_attention(C.byref(d) if d is not None else None, q, s, heads, lengths, 1.0, window, out, s, None, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_bad_caches_are_refused_by_both_calls(bad):
    d = _desc(**bad)
    assert _append(d) == INVALID
    assert lib.load().gcb200_last_error().startswith(b"paged")
    assert _attend(d) == INVALID
    assert lib.load().gcb200_last_error().startswith(b"paged")


def test_overlapping_cache_rows_are_refused_where_they_would_be_written():
    d = _desc(key_stride=(2048, 0, 64))
    assert _append(d) == INVALID


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(pos=None), dict(out=None), dict(tokens=-1), dict(heads=0), dict(tokens=4),
                                 dict(rotary=64), dict(inv=P), dict(inv=P, rotary=63), dict(inv=P, rotary=66)])
def test_append_refuses(bad):
    assert _append(_desc(), **bad) == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(lengths=None), dict(ws=None), dict(ws=P + 8), dict(ws_bytes=0), dict(heads=3), dict(heads=0),
                                 dict(window=-1)])
def test_attention_refuses(bad):
    assert _attend(_desc(), **bad) == INVALID


def test_empty_calls_and_null_descriptors():
    assert _append(None) == INVALID and _attend(None) == INVALID
    assert _append(_desc(), tokens=0, q=None, k=None, v=None, pos=None) == OK      # nothing to do, no device needed
    assert _append(_desc(sequences=0, page_table=None), tokens=0) == OK


def test_w4_sizes_and_refusals():
    l, n = lib.load(), C.c_size_t(0)

    def size(N, K, g, z):
        st = l.gcb200_w4_packed_bytes(N, K, g, z, C.byref(n))
        return n.value if st == OK else -st

    assert size(16, 128, 128, 0) == 1024 + 32 and size(17, 129, 128, 1) == 4 * (1024 + 32 + 16)
    assert size(16, 128, 64, 1) == 1024 + 64 + 32 and size(16, 128, 32, 0) == 1024 + 128 and size(16, 256, 256, 0) == 2 * (1024 + 32)
    for bad in [(0, 128, 128), (16, 0, 128), (16, 128, 0), (16, 128, 16), (16, 128, 96), (16, 128, 200), (16, 128, -128)]:
        assert size(*bad, 0) == -INVALID
    mm = l.gcb200_matmul_w4
    good = [BF16, P, 128, P, None, P, 16, 2, 16, 128, 128, 0, 0, None]
    for i, v in [(0, 3), (0, E4M3), (1, None), (3, None), (5, None), (3, P + 8), (2, 127), (6, 15), (7, -1), (8, 0), (9, 0), (10, 48)]:
        args = list(good)
        args[i] = v
        assert mm(*args) == INVALID, (i, v)
    args = list(good)
    args[7] = 0
    assert mm(*args) == OK       # no rows: nothing to do
    assert l.gcb200_w4_pack(None, 64, P, 1, None, 0, 16, 128, 128, P, None) == INVALID
    assert l.gcb200_w4_pack(P, 64, P, 1, None, 0, 16, 128, 128, P + 4, None) == INVALID


HARNESS = r"""
#include "paged_index.h"
extern "C" int t_page_of(const int32_t *e, int64_t stride, int sequences, int max_pages, int page_size, int pages, int seq, int pos) {
  gcb::PageTable t{e, stride, sequences, max_pages, page_size, pages};
  return gcb::page_of(t, seq, pos);
}
extern "C" void t_seen_of(int max_pages, int page_size, int length, int window, int *out) {
  gcb::PageTable t{nullptr, 0, 1, max_pages, page_size, 1};
  gcb::Seen s = gcb::seen_of(t, length, window);
  out[0] = s.first; out[1] = s.end; out[2] = s.cut;
}
extern "C" int64_t t_share_of(int64_t total, int blocks, int least) { return gcb::share_of(total, blocks, least); }
extern "C" int64_t t_part_slot(int64_t block, int64_t per, int64_t begin) { return gcb::part_slot(block, per, begin); }
extern "C" int t_first_cut(int64_t i, int64_t per, int64_t begin, int64_t end) { return gcb::first_cut(i, per, begin, end); }
extern "C" int t_tiles_of(int first, int end, int tile) { return gcb::tiles_of(gcb::Seen{first, end, false}, tile); }
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("index")
    (d / "h.cpp").write_text(HARNESS)
    so = d / "h.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "graph-compiler_b200", "csrc"), str(d / "h.cpp"), "-o", str(so)], check=True)
    l = C.CDLL(str(so))
    l.t_page_of.argtypes = [C.c_void_p, C.c_int64] + [C.c_int] * 6
    l.t_seen_of.argtypes = [C.c_int] * 4 + [C.c_void_p]
    for name, args in (("t_share_of", [C.c_int64, C.c_int, C.c_int]), ("t_part_slot", [C.c_int64] * 3), ("t_first_cut", [C.c_int64] * 4)):
        getattr(l, name).argtypes = args
    l.t_share_of.restype = l.t_part_slot.restype = C.c_int64
    return l


def test_bad_pages_are_never_followed(index):
    table = np.array([[3, -1, 7, 8, 99], [0, 2147483647, -2147483648, 5, 99]], dtype=np.int32)   # the last column belongs to no row

    def page(seq, pos, pages=8):
        return index.t_page_of(table.ctypes.data, 5, 2, 4, 6, pages, seq, pos)

    assert [page(0, p) for p in (0, 5, 6, 12, 17, 18, 23)] == [3, 3, -1, 7, 7, -1, -1]
    assert [page(1, p) for p in (0, 6, 12, 18)] == [0, -1, -1, 5]
    assert [page(0, p) for p in (24, 29, 2147483647, -1, -2147483648)] == [-1] * 5     # no entry for these positions
    assert page(2, 0) == -1 and page(-1, 0) == -1 and page(2147483647, 0) == -1        # no such sequence
    assert page(0, 0, pages=3) == -1 and page(0, 0, pages=4) == 3


def test_seen_positions(index):
    out = (C.c_int * 3)()

    def seen(length, window, max_pages=4, page_size=6):
        index.t_seen_of(max_pages, page_size, length, window, out)
        return tuple(out)

    assert seen(0, 0) == (0, 0, 0) and seen(-5, 3) == (0, 0, 0) and seen(-2147483648, 1) == (0, 0, 0)
    assert seen(7, 0) == (0, 7, 0) and seen(7, 7) == (0, 7, 0) and seen(7, 8) == (0, 7, 0) and seen(7, 2) == (5, 7, 0)
    assert seen(24, 0) == (0, 24, 0) and seen(25, 0) == (0, 24, 1) and seen(2147483647, 1) == (23, 24, 1)
    assert seen(3, 0, max_pages=0) == (0, 0, 1)


@pytest.mark.parametrize("seed", range(60))
def test_every_tile_has_one_block_and_every_cut_unit_one_join(index, seed):
    """The blocks' shares, walked as the kernel walks them: each tile once, no more than two parts to a block, and the parts that
    the join of a cut unit reads are those that were written for it."""
    r = np.random.RandomState(seed)
    tile, units, blocks, least = int(r.choice([64, 128])), int(r.choice([1, 2, 8, 40])), int(r.choice([1, 2, 7, 148, 592])), int(r.choice([1, 1, 2, 5]))
    lengths = [int(x) for x in r.randint(0, r.choice([2, 100, 3000]), r.choice([1, 3, 50]))]
    begins, at = [], 0
    for n in lengths:
        k = index.t_tiles_of(0, n, tile)
        assert k == -(-n // tile)
        begins += [(at + u * k, at + (u + 1) * k) for u in range(units) if k]
        at += k * units
    total, per = at, index.t_share_of(at, blocks, least)
    assert per >= least and per * blocks >= total
    written, whole = {}, set()
    for b in range(blocks):
        lo, hi = b * per, min(total, (b + 1) * per)
        for u, (x, y) in enumerate(begins):
            if max(lo, x) < min(hi, y):
                if lo <= x and y <= hi:
                    whole.add(u)
                else:
                    slot = 2 * b + (1 if x >= lo else 0)
                    assert slot not in written and slot < 2 * blocks
                    written[slot] = u
    joined = set()
    for i in range(1, blocks):
        if i * per >= total:
            continue
        u = next(k for k, (x, y) in enumerate(begins) if x <= i * per < y)
        x, y = begins[u]
        if index.t_first_cut(i, per, x, y):
            assert u not in joined
            joined.add(u)
            slots = [index.t_part_slot(b, per, x) for b in range(x // per, (y - 1) // per + 1)]
            assert len(slots) > 1 and all(written[s] == u for s in slots)
            assert slots == [s for s in sorted(written) if written[s] == u]
    assert joined == set(written.values()) and not joined & whole and len(joined) + len(whole) == len(begins)
