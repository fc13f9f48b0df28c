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
