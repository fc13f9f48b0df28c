"""Refusals of the decode operators without a device: results whose rows overlap, on which several thread blocks would write at once."""
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
