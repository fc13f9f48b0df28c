"""Attention over the paged cache where results are small beside what they are summed from: what the weights of the softmax lose on
their way into the product with the values would show.

Tokens come in pairs of almost the same key and opposite values.  With A the largest sum of |q k| scale, n tokens:
  result    rounded once: u |o| (bf16 2^-8, f16 2^-11)
  scores    dim / 16 products of sixteen, each sum off by 2^-22 of its terms at most, then two roundings: (dim / 16 + 2) 2^-22 A
  weights   2^-22 of the exponential itself; held to 2^-15 + 2^-20 in bf16 (the rest behind eight bits is below 2^-7, eight bits of it
            are kept) and to 2^-21 in f16, where numbers below its normal range add 2^-23 of a unit that the largest weight is 2^7 of;
            bf16 results over an 8-bit cache: one f16 number, half a step of which is 2^-11
  sums      n / 16 products of sixteen: (n / 16 + 2) 2^-22; the softmax's own sum the same
and the scores' and weights' parts count twice, for the sum that they are divided by."""
import pytest
import torch

from gc_b200 import lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("heads,kv", [(4, 2), (8, 1), (16, 1)])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("length", [2, 64, 5000])
def test_weights_keep_their_bits(dtype, cache, heads, kv, dim, length):
    g = torch.Generator(device="cuda").manual_seed(dim + heads + length)
    page, f8 = 16, cache == torch.float8_e4m3fn
    raw = torch.uint8 if f8 else torch.int16
    pages = -(-length // page)
    k = (1 + torch.rand(pages * page // 2, kv, dim, generator=g, device="cuda")).to(cache)      # one binade: a step is the same everywhere
    other = k.clone()
    other.view(raw)[:, :, 0] ^= 1                                                               # a step up or down in one place
    v = (torch.randn(pages * page // 2, kv, dim, generator=g, device="cuda")).to(cache)
    tokens = lambda a, b: torch.stack([a.view(raw), b.view(raw)], 1).flatten(0, 1).view(cache)  # noqa: E731
    key, value = tokens(k, other), tokens(v, (-v.float()).to(cache))
    paged = lambda t: t.view(raw).view(pages, page, kv, dim).transpose(1, 2).view(cache)        # noqa: E731
    q = (torch.rand(1, heads, dim, generator=g, device="cuda") / 2 + 0.5).to(dtype)
    q[..., 1:] *= torch.where(torch.rand(dim - 1, generator=g, device="cuda") < 0.5, -1.0, 1.0).to(dtype)
    scale = 1.0 / dim
    ones = torch.ones(kv, device="cuda") if f8 else None
    out = lib.paged_attention(q, paged(key), paged(value), torch.arange(pages, dtype=torch.int32, device="cuda")[None],
                              torch.tensor([length], dtype=torch.int32, device="cuda"), scale, key_scale=ones, value_scale=ones)[0].double()
    kd, vd = (t[:length].double().transpose(0, 1).repeat_interleave(heads // kv, 0) for t in (key, value))   # [heads, n, dim]
    x = torch.einsum("hd,hnd->hn", q[0].double(), kd) * scale
    A = float(torch.einsum("hd,hnd->hn", q[0].double().abs(), kd.abs()).max()) * scale
    assert A <= 2
    p = torch.softmax(x, -1)[:, None]
    want, mag, top = (p @ vd)[:, 0], (p @ vd.abs())[:, 0], vd.abs().amax()
    f16 = f8 or dtype == torch.float16
    weights = (dim / 16 + 2) * 2.0 ** -22 * A + 2.0 ** -22 + (2.0 ** -11 if f8 and dtype == torch.bfloat16 else 2.0 ** -21 if f16 else 2.0 ** -15 + 2.0 ** -20)
    tol = U[dtype] * want.abs() + (2 * weights + 2 * (length / 16 + 2) * 2.0 ** -22) * mag + (length * 2.0 ** -30 * top if f16 else 0) + 2.0 ** -24
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())
    assert lib.device_error() == 0
