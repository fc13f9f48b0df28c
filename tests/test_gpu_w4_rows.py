"""4-bit linear layers: any number of rows, and rows that do not depend on one another.

A result is off by at most u |y| (one rounding; bf16 2^-8, f16 2^-11) and 2^-14 sum |x| |w|: products are exact in f32, and at most 2^9
f32 additions follow one another."""
import pytest
import torch

from gc_b200 import lib

pytestmark = pytest.mark.gpu

T, U = {"bf16": torch.bfloat16, "f16": torch.float16}, {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _layer(N, K, group, dtype, seed, zeros=False):
    """(packed weights, W in 64 bits on the device)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-K // group)
    codes = torch.randint(0, 256, (N, (K + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand(N, groups, generator=g, device="cuda")).to(T[dtype])
    zs = torch.randint(0, 16, (N, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    w = torch.stack([codes & 15, codes >> 4], -1).flatten(1)[:, :K].double()
    spread = lambda t: t.double().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    return lib.pack_w4(codes, scales, K, group, zeros=zs), (w - (8 if zs is None else spread(zs))) * spread(scales)


def _check(y, x, w, dtype):
    for i in range(0, x.shape[0], 65536):
        xs, got = x[i:i + 65536].double(), y[i:i + 65536].double()
        want = xs @ w.T
        assert ((got - want).abs() <= U[dtype] * want.abs() + 2.0 ** -14 * (xs.abs() @ w.abs().T)).all()


@pytest.mark.parametrize("M,dtype", [(8 * 65535 + 1, "bf16"), (16 * 65535, "f16"), (16 * 65535 + 1, "bf16"), (2 * 16 * 65535 + 17, "f16")])
def test_more_rows_than_a_grid_has_passes(M, dtype):
    p, w = _layer(24, 40, 32, dtype, 0, zeros=True)
    x = torch.randn(M, 40, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(T[dtype])
    whole = torch.full((M + 1, 26), 3.0, dtype=T[dtype], device="cuda")
    lib.matmul_w4(x, p, out=whole[:M, :24])
    _check(whole[:M, :24], x, w, dtype)
    assert (whole[M:] == 3).all() and (whole[:, 24:] == 3).all()
    assert lib.device_error() == 0


@pytest.mark.parametrize("M,N,K,group,dtype", [(16, 4096, 2048, 128, "bf16"), (13, 1000, 4095, 32, "f16"), (40, 333, 384, 64, "bf16"), (5, 48, 30000, 128, "f16")])
def test_rows_of_a_call_and_rows_alone(M, N, K, group, dtype):
    """Each row computed alone is right by itself, and within both calls' bounds of its result among the others (bits may differ: the
    work is shared out by the number of rows)."""
    p, w = _layer(N, K, group, dtype, M)
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(T[dtype])
    y = lib.matmul_w4(x, p)
    _check(y, x, w, dtype)
    alone = torch.cat([lib.matmul_w4(x[m:m + 1], p) for m in range(M)])
    _check(alone, x, w, dtype)
    assert lib.device_error() == 0


def test_calls_on_several_streams_at_once():
    """Different layers under way on four streams, one synchronisation at the end: each result has the bits of the call made alone."""
    sizes = [(1, 4096, 4096, 128), (16, 2048, 8192, 128), (3, 11001, 1030, 32), (9, 64, 60000, 64)]
    layers = [_layer(N, K, group, "bf16", i)[0] for i, (_, N, K, group) in enumerate(sizes)]
    xs = [torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").bfloat16() for i, (M, _, K, _) in enumerate(sizes)]
    want = [lib.matmul_w4(x, p) for x, p in zip(xs, layers)]
    outs = [[torch.empty_like(w) for _ in range(8)] for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    for k in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                lib.matmul_w4(xs[(i + k) % 4], layers[(i + k) % 4], out=outs[(i + k) % 4][k])
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os, w in zip(outs, want) for o in os)
    assert lib.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_infinities_and_nan_make_their_rows_nan(dtype, zeros):
    p, w = _layer(96, 200, 32, dtype, 3, zeros=zeros)
    x = torch.randn(5, 200, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(T[dtype])
    clean = lib.matmul_w4(x, p)
    x[1, 7], x[2, 199], x[3, 0] = float("nan"), float("inf"), -float("inf")
    for relu in (False, True):
        y = lib.matmul_w4(x, p, relu=relu)
        assert y[1:4].isnan().all()
        for m in (0, 4):
            assert torch.equal(y[m], clean[m].clamp(min=0) if relu else clean[m])
