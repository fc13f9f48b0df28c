"""Attention over long sequences of one KV head: a softmax in a hundred parts, which the join reads in several turns.

The result is rounded once: u |o|; the exponentials are rounded to the 16-bit type of the product with the values: u_p sum p |v| / sum p;
scores of f32 and the exponentials' own error 2^-13 together (magnitudes of the scores stay below 2^6).  Sums of 2^15 terms in f32, added
up in turns of less than 2^10, add 2^-14."""
import math

import pytest
import torch

from gc_b200 import lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("dim,heads", [(256, 3), (256, 9), (144, 8), (128, 16), (64, 40)])
@pytest.mark.parametrize("length", [6001, 30011])
def test_many_parts(dtype, cache, dim, heads, length):
    g = torch.Generator(device="cuda").manual_seed(length + dim)
    page = 16
    per = -(-length // page)
    table = torch.randperm(per + 1, generator=g, device="cuda")[:per].to(torch.int32)[None]
    f8 = cache == torch.float8_e4m3fn
    keys, values = ((torch.randn(per + 1, 1, page, dim, generator=g, device="cuda") * (30 if f8 else 1)).to(cache) for _ in range(2))
    ks, vs = (torch.tensor([x], device="cuda") if f8 else None for x in (0.03, 0.05))
    q = (torch.randn(1, heads, dim, generator=g, device="cuda") * 1.5).to(dtype)
    lse = torch.empty(1, heads, device="cuda")
    out = lib.paged_attention(q, keys, values, table, torch.tensor([length], dtype=torch.int32, device="cuda"), dim ** -0.5, key_scale=ks, value_scale=vs, lse=lse)
    k = keys[table[0].long(), 0].double().flatten(0, 1)[:length] * (ks.double() if f8 else 1)
    v = values[table[0].long(), 0].double().flatten(0, 1)[:length] * (vs.double() if f8 else 1)
    x = q[0].double() @ k.T * dim ** -0.5
    assert x.abs().max() < 64
    p = torch.softmax(x, -1)
    want, mag = p @ v, p @ v.abs()
    up = 2.0 ** -11 if f8 else U[dtype]
    assert ((out[0].double() - want).abs() <= U[dtype] * want.abs() + (up + 2.0 ** -13 + 2.0 ** -14) * mag + 1e-7).all()
    assert ((lse[0].double() - torch.logsumexp(x, -1)).abs() <= 2.0 ** -13 + 2.0 ** -14 + 2.0 ** -20 * math.log(length)).all()
    assert lib.device_error() == 0
