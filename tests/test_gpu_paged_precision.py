"""Attention over the paged cache where results are small beside what they are summed from: what the weights of the softmax lose on
their way into the product with the values would show.

Tokens come in pairs of almost the same key and opposite values.  With A the largest sum of |q k| scale, n tokens:
  result    rounded once: u |o| (bf16 2^-8, f16 2^-11)
  scores    dim / 16 products of sixteen, each sum off by 2^-22 of its terms at most, then two roundings: (dim / 16 + 2) 2^-22 A
  weights   2^-22 of the exponential itself; held to 2^-15 + 2^-20 in bf16 (the rest behind eight bits is below 2^-7, eight bits of it
            are kept) and to 2^-20 in f16 (the rest is below 2^-9), where numbers below its normal range add 2^-23 of a unit that the largest
            weight is 2^7 of;
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
    weights = (dim / 16 + 2) * 2.0 ** -22 * A + 2.0 ** -22 + (2.0 ** -11 if f8 and dtype == torch.bfloat16 else 2.0 ** -20 if f16 else 2.0 ** -15 + 2.0 ** -20)
    tol = U[dtype] * want.abs() + (2 * weights + 2 * (length / 16 + 2) * 2.0 ** -22) * mag + (length * 2.0 ** -30 * top if f16 else 0) + 2.0 ** -24
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())
    assert lib.device_error() == 0


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn), (torch.float16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("bits", [8, 16, 21, 25])
@pytest.mark.parametrize("heads", [1, 16])
def test_many_light_tokens(dtype, cache, bits, heads):
    """A few tokens of value zero, one for each part of a tile, and twenty thousand of value one with about 2^-bits of a weight each, in so
    many sequences that a block has a whole one.  A weight is off by 2^-24 of a unit that the largest is 2^7 of, at most, and to
    either side: over all, at 2^-25 of the largest, 2^-7 / sqrt(3 n) of the result, eight times which is 2^-11.9.  Sums, scores of f32 and
    exponentials: 2^-12.  A bias of 2^-24 of that unit would be 2^-6."""
    g = torch.Generator(device="cuda").manual_seed(bits)
    n, dim, page, f8, sequences = 20000, 16, 32, cache == torch.float8_e4m3fn, 600
    raw = torch.uint8 if f8 else torch.int16
    pages = n // page
    k = -(1 + torch.randint(0, 8, (n, 1, dim), generator=g, device="cuda") / 8.0)
    v = torch.ones(n, 1, dim, device="cuda")
    k[:128:16], v[:128:16] = 0, 0
    paged = lambda t: t.to(cache).view(raw).view(pages, page, 1, dim).transpose(1, 2).view(cache)   # noqa: E731
    q = (bits * 0.6931 / (dim * 1.4375) * (0.9 + 0.2 * torch.rand(sequences, heads, dim, generator=g, device="cuda"))).to(dtype)
    ones = torch.ones(1, device="cuda") if f8 else None
    out = lib.paged_attention(q, paged(k), paged(v), torch.arange(pages, dtype=torch.int32, device="cuda").repeat(sequences, 1),
                              torch.full((sequences,), n, dtype=torch.int32, device="cuda"), 1.0, key_scale=ones, value_scale=ones).double()
    w = torch.exp(q.double() @ k[:, 0].double().T)
    want = (w @ v[:, 0].double()) / w.sum(-1, keepdim=True)
    tol = (U[dtype] + 2.0 ** -10.9) * want
    assert ((out - want).abs() <= tol).all(), float(((out - want).abs() / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 8, 16])
def test_infinite_values_give_infinite_results(dtype, heads):
    """Whatever a weight is, its two parts are of one sign where an infinity meets them, and neither is zero."""
    g = torch.Generator(device="cuda").manual_seed(heads)
    n, dim = 64, 64
    k = torch.randn(4, 1, 16, dim, generator=g, device="cuda").to(dtype)
    v = torch.randn(4, 1, 16, dim, generator=g, device="cuda").to(dtype)
    for t in range(n):
        v[t // 16, 0, t % 16, t % dim] = float("inf") if t % 2 else -float("inf")
    k[0, 0, 3] = 0      # with queries of zeros for head 0: weights of exactly one
    q = (torch.randn(1, heads, dim, generator=g, device="cuda") * 0.5).to(dtype)
    q[0, 0] = 0
    out = lib.paged_attention(q, k, v, torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda"), dim ** -0.5)
    sign = torch.where(torch.arange(dim, device="cuda") % 2 == 1, float("inf"), -float("inf"))
    assert (out[0].float() == sign).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [1, 10, 13, 14, 15, 20, 22, 28])
def test_an_infinite_value_of_a_light_token(dtype, bits):
    """Down to 2^-28 of the largest weight."""
    k, v = torch.zeros(1, 1, 16, 16, device="cuda", dtype=dtype), torch.ones(1, 1, 16, 16, device="cuda", dtype=dtype)
    k[0, 0, 1, 0], v[0, 0, 1, 3], v[0, 0, 1, 4] = -bits, float("inf"), -float("inf")
    q = torch.zeros(1, 3, 16, device="cuda", dtype=dtype)
    q[0, :, 0] = torch.tensor([1.0, 0.9375, 0.875])
    out = lib.paged_attention(q, k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([2], dtype=torch.int32, device="cuda"), 0.6931472)
    assert (out[0, :, 3] == float("inf")).all() and (out[0, :, 4] == -float("inf")).all() and out[0, :, :3].isfinite().all() and out[0, :, 5:].isfinite().all()
