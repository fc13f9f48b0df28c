"""How a call of the 4-bit linear layer is shared out (compiled here for the host): whatever the sizes, the pieces in shared memory
are as large as the kernel's own arithmetic needs, and lie one behind the other."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HARNESS = r"""
#include "w4_plan.h"
extern "C" int t_plan(int M, int tiles, int kblocks, int64_t group, int zeros, const int *at_once, int *out) {
  gcb::W4Plan p{};
  if (!gcb::plan_w4(M, tiles, kblocks, gcb::groups_per_block(group), gcb::block_bytes(group, zeros != 0), at_once, &p)) return 0;
  const int v[13] = {p.pass, p.nt, p.rt, p.cluster, p.share, p.wk, p.clusters, p.stages, p.x_at, p.table_at, p.meet_at, p.part_at, p.smem};
  for (int i = 0; i < 13; ++i) out[i] = v[i];
  return 1;
}
"""
AT_ONCE = (C.c_int * 9)(0, 148, 74, 0, 33, 0, 0, 0, 14)
MOST = 223 * 1024


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "h.cpp").write_text(HARNESS)
    so = d / "h.so"
    subprocess.run(["g++", "-O1", "-fwrapv", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "graph-compiler_b200", "csrc"), str(d / "h.cpp"), "-o", str(so)], check=True)
    l = C.CDLL(str(so))
    l.t_plan.argtypes = [C.c_int] * 3 + [C.c_int64, C.c_int, C.c_void_p, C.c_void_p]

    def call(M, N, K, group, zeros):
        out = (C.c_int * 13)()
        if not l.t_plan(M, -(-N // 16), -(-K // 128), group, zeros, AT_ONCE, out):
            return None
        return dict(zip("pass_ nt rt cluster share wk clusters stages x_at table_at meet_at part_at smem".split(), out))

    return call


def _check(p, M, N, K, group, zeros):
    gpb = 1 if group >= 128 else 128 // group
    tiles, kblocks, block = -(-N // 16), -(-K // 128), 1024 + gpb * 16 * (3 if zeros else 2)
    assert 1 <= p["pass_"] <= min(M, 16) and p["nt"] == (2 if p["pass_"] > 8 else 1) and p["rt"] in (1, 2)
    assert p["cluster"] in (1, 2, 4, 8) and 1 <= p["clusters"] <= min(AT_ONCE[p["cluster"]], tiles)
    assert p["wk"] in (1, 2, 4, 8, 16) and 2 <= p["stages"] <= 4
    assert p["share"] * p["cluster"] >= kblocks
    outs = 16 * p["rt"] * (16 // p["wk"])
    rows = p["pass_"] + 1
    pieces = [("ring", 0, 16 * p["stages"] * p["rt"] * block, p["x_at"]), ("x", p["x_at"], rows * (p["share"] * 256 + 64), p["table_at"]),
              ("table", p["table_at"], p["share"] * gpb * rows * 8, p["meet_at"]),
              ("meet", p["meet_at"], 16 * 8 * p["nt"] * (16 * p["rt"] + 4) * 4, p["part_at"]),
              ("part", p["part_at"], 2 * 8 * p["nt"] * outs * 4 if p["cluster"] > 1 else 0, p["smem"])]
    for name, at, need, end in pieces:
        assert at % 16 == 0 and at + need <= end <= MOST, (name, at, need, end)


# rows of x whose bytes, and those with the table behind them, pass 2^31 and 2^32
LONG = [(M, 128 * c * (w // ((min(M, 16) + 1) * per) + d)) for M in (1, 4, 8, 16) for c in (1, 2, 4, 8) for w in (2 ** 31, 2 ** 32, 2 ** 33, 2 ** 34)
        for per in (256, 264, 272, 288) for d in (-3, -1, 0, 1, 2, 20, 200)]


@pytest.mark.parametrize("group,zeros", [(32, 1), (64, 0), (128, 0)])
def test_rows_that_fit_into_no_cluster_are_refused(plan, group, zeros):
    for M, K in [(16, 1 << 26), (1, 195585), (1, 260000), (7, (1 << 31) - 1)] + [x for x in LONG if 195584 < x[1] < 2 ** 31]:
        assert plan(M, 64, K, group, zeros) is None, (M, K)


@pytest.mark.parametrize("seed", range(8))
def test_pieces_of_shared_memory(plan, seed):
    r = np.random.RandomState(seed)
    for _ in range(400):
        M, N, K = int(2 ** r.uniform(0, 19)), int(2 ** r.uniform(0, 31)) - 1 or 1, int(2 ** r.uniform(0, 17.6))
        K, group, zeros = min(K, 195584), int(r.choice([32, 64, 128, 1024])), int(r.randint(2))
        p = plan(M, N, K, group, zeros)
        assert p is not None, (M, N, K, group, zeros)
        _check(p, M, N, K, group, zeros)


def test_rows_of_x_to_a_pass(plan):
    """What the header says about the rows that read the weights once."""
    for K, rows in [(22528, 16), (22529, 8), (43008, 8), (43009, 4), (77824, 4), (77825, 2), (130048, 2), (130049, 1), (195584, 1)]:
        for group, zeros in ((32, 1), (64, 1), (128, 0)):
            assert plan(16, 4096, K, group, zeros)["pass_"] == rows, (K, group)
