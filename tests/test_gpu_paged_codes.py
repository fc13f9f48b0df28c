"""What an 8-bit cache holds of a new value: x / scale in f32 (a quotient of a division, rounded once), limited, to the nearest code.
The same arithmetic on the CPU gives the same bits."""
import pytest
import torch

from gc_b200 import lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (48, 24), (16, 6)])     # eight elements at a time, four, and single ones
@pytest.mark.parametrize("scale", [1.0, 3.0, 1.0 / 3.0, 0.1, 7.0, 0.0234375, 1.25e-3, 1.1754944e-38 * 2 ** 20, 5.0e20])
def test_every_number_by_a_scale(dtype, dim, rotary, scale):
    """All 65536 numbers of the type as values, through a call that rotates its keys by nothing."""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    tokens = -(-65536 // dim)
    x = torch.cat([x, x[:tokens * dim - 65536]]).view(tokens, 1, dim)
    page = 64
    pages = -(-tokens // page)
    keys, values = (torch.zeros(pages, 1, page, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    scales = torch.tensor([scale], dtype=torch.float32)
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda")
    lib.paged_kv_append(None, x.cuda(), x.cuda(), keys, values, torch.arange(pages, dtype=torch.int32, device="cuda")[None], pos, sequences=torch.zeros_like(pos),
                        inv_freq=torch.zeros(rotary // 2, dtype=torch.float64, device="cuda"), key_scale=scales.cuda(), value_scale=scales.cuda())
    want = (x.float() / scales).clamp(-448, 448).to(torch.float8_e4m3fn).view(tokens, dim).float()
    got = values.view(torch.uint8)[:, 0].flatten(0, 1)[:tokens].view(torch.float8_e4m3fn).float().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num()), int((got.nan_to_num() != want.nan_to_num()).sum())
    assert lib.device_error() == 0
