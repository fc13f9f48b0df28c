"""Refusals of the decode operators without a device: results whose rows overlap, on which several thread blocks would write at once, and addresses at which
a kernel would stop with a fault."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from gc_b200 import lib
from test_decode_host import INVALID, P, _desc, _i64s

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "h.cpp").write_text('#include "paged_index.h"\nextern "C" int t(int64_t na, int64_t a, int64_t nb, int64_t b, int64_t dim) { return gcb::rows_overlap(na, a, nb, b, dim); }\n')
    so = d / "h.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "graph-compiler_b200", "csrc"), str(d / "h.cpp"), "-o", str(so)], check=True)
    l = C.CDLL(str(so))
    l.t.argtypes = [C.c_int64] * 5
    return lambda *a: bool(l.t(*a))


def test_rows_overlap_where_they_do(overlap):
    r = np.random.RandomState(0)
    seen = set()
    for _ in range(4000):
        na, nb, dim = int(r.randint(0, 7)), int(r.randint(0, 7)), int(r.randint(1, 6))
        a, b = int(r.randint(-40, 40)), int(r.randint(-40, 40))
        if r.rand() < 0.3:
            b = a * max(na, 1) + int(r.randint(-1, 2))
        at = [i * a + j * b + e for i in range(na) for j in range(nb) for e in range(dim)]
        want = len(set(at)) < len(at)
        assert overlap(na, a, nb, b, dim) == want, (na, a, nb, b, dim)
        seen.add(want)
    assert seen == {False, True}
    assert not overlap(1 << 30, 64, 65535, 64 << 30, 64) and overlap(1 << 30, 64, 2, (64 << 30) - 64, 64)


@pytest.mark.parametrize("stride", [(0, 64), (256, 0), (256, 63), (64, 64), (192, 64)])
def test_results_whose_rows_overlap_are_refused(stride):
    l, d, s, o = lib.load(), _desc(), _i64s(256, 64), _i64s(*stride)
    assert l.gcb200_paged_attention(C.byref(d), P, s, 4, P, 1.0, 0, P, o, None, P, 1 << 30, None) == INVALID
    assert b"overlap" in l.gcb200_last_error()
    assert l.gcb200_paged_kv_append(C.byref(d), P, s, 4, P, s, P, s, P, o, None, P, 3, None, 0, 0, None) == INVALID
    assert b"overlap" in l.gcb200_last_error()


def test_misaligned_addresses_are_refused():
    l, s, n = lib.load(), _i64s(256, 64), 0
    attend = [P, s, 4, P, 1.0, 0, P, s, P, P, 1 << 30, None]
    append = [P, s, 4, P, s, P, s, P, s, P, P, 3, P, 64, 0, None]
    matmul = [2, P, 128, P, P, P, 16, 2, 16, 128, 128, 0, 0, None]
    descs = [_desc(page_table=P + 2), _desc(cache_dtype=10, key_scale=P + 1), _desc(cache_dtype=10, value_scale=P + 2)]
    for d in descs:
        assert l.gcb200_paged_attention(C.byref(d), *attend) == INVALID and l.gcb200_paged_kv_append(C.byref(d), *append) == INVALID
    for call, good, at in ((l.gcb200_paged_attention, [C.byref(_desc())] + attend, {1: 1, 4: 2, 7: 1, 9: 2}),
                           (l.gcb200_paged_kv_append, [C.byref(_desc())] + append, {1: 1, 4: 1, 6: 1, 8: 1, 10: 2, 11: 2, 13: 4}),
                           (l.gcb200_matmul_w4, matmul, {1: 1, 4: 1, 5: 1})):
        for i, off in at.items():
            assert good[i] == P
            assert call(*good[:i], P + off, *good[i + 1:]) == INVALID, (call.__name__, i)
            assert b"misaligned" in l.gcb200_last_error()
            n += 1
    assert n == 14
