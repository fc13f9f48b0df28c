"""What a bad page number or length leaves behind: a code that the program can read, and nothing that another call takes for a
failure of its own."""
import numpy as np
import pytest
import torch

import oracle
from _util import assert_bf16_close, tbits
from gc_b200 import api, lib, partitions, tune
from gc_b200 import benchgc_compat as bc

pytestmark = pytest.mark.gpu


def _attend(page):
    """Two sequences of 64 tokens; the first one's second page is `page`."""
    g = torch.Generator().manual_seed(0)
    keys, values = (torch.randn(8, 2, 16, 64, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(2, 4, 64, generator=g).bfloat16().cuda()
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    table[0, 1] = page
    return lib.paged_attention(q, keys, values, table.cuda(), torch.tensor([64, 64], dtype=torch.int32).cuda(), 0.125)


def _append(page):
    x, cache = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    lib.paged_kv_append(None, x, x, cache, cache.clone(), torch.tensor([[page]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda())


@pytest.mark.parametrize("call", [_attend, _append])
def test_a_bad_page_does_not_fail_the_next_execute(call):
    assert lib.device_error() == 0
    A = bc.fill_tensor((128, 512), "bf16", "U", (-1, 1), 0)
    W = bc.fill_tensor((512, 256), "bf16", "U", (-1, 1), 1)
    b = bc.fill_tensor((256,), "bf16", "U", (-1, 1), 2)
    js, _, out_id = partitions.mlp(128, (512, 256), "bf16", [True], "relu")
    want, acc = oracle.linear_bf16(tbits(A), tbits(W), tbits(b), relu=True, return_acc=True)
    exe = api.GraphCompiler().compile(js)
    out = torch.empty(128, 256, dtype=torch.bfloat16)
    call(99)
    torch.cuda.synchronize()
    exe.execute({0: A, 1: W, 2: b}, {out_id: out})
    assert_bf16_close(tbits(out), want, 512, what="behind a call with a bad page", pre=acc)
    assert lib.device_error() == 9 and lib.device_error() == 0     # and the program still learns of it, once


@pytest.mark.parametrize("page_first", [False, True])
def test_a_bad_page_and_a_wait_that_ran_out_are_both_reported(page_first):
    assert lib.device_error() == 0
    for page in (page_first, not page_first):
        _attend(-5) if page else lib.wait_selftest(200_000)
    assert lib.device_error() == 7 and lib.device_error() == 9 and lib.device_error() == 0


def test_wait_error_leaves_a_bad_page():
    _attend(8)
    assert lib.wait_error() == 0
    lib.wait_selftest(200_000)
    assert lib.wait_error() == 7 and lib.wait_error() == 0 and lib.device_error() == 9 and lib.device_error() == 0


def test_tuning_behind_a_bad_page():
    _attend(8)
    M, N, K = 16, 512, 256
    tune.tune_matmul(M, N, K, iters=2, record=False)
    assert lib.device_error() == 9


def test_a_long_row_of_bad_pages():
    """Every token's page is bad: they all count as zeros, and the call is reported."""
    S, H, D, page, n = 2, 8, 128, 16, 16384
    keys = torch.ones(1, H, page, D, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(S, H, D, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    table = torch.full((S, n // page), -1, dtype=torch.int32, device="cuda")
    lens, lse = torch.full((S,), n, dtype=torch.int32, device="cuda"), torch.empty(S, H, device="cuda")
    out = lib.paged_attention(q, keys, keys, table, lens, 1.0, lse=lse)
    assert lib.device_error() == 9 and lib.device_error() == 0
    assert not out.any() and np.allclose(lse.cpu().numpy(), np.log(n), rtol=0, atol=2.0 ** -19)


def _us(call, n=5):
    call()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(n):
        call()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / n * 1e3


def test_bad_pages_and_lengths_cost_no_more_than_good_ones():
    """The code is recorded in host memory; a wait for the host at every token, sequence or thread would take 5000 times as long.  The
    bound leaves room for a loaded host: the good calls take 20 to 100 us."""
    g = torch.Generator(device="cuda").manual_seed(0)
    H, D, page, n = 8, 128, 16, 16384
    keys = torch.randn(2 * n // page, H, page, D, device="cuda", generator=g).bfloat16()
    q, lens = torch.randn(2, H, D, device="cuda", generator=g).bfloat16(), torch.full((2,), n, dtype=torch.int32, device="cuda")
    good = torch.arange(2 * n // page, dtype=torch.int32, device="cuda").view(2, -1)
    bad = torch.full_like(good, -1)
    attend = [_us(lambda: lib.paged_attention(q, keys, keys, t, lens, 1.0)) for t in (good, bad)]

    x, other = torch.randn(n, H, D, device="cuda", generator=g).bfloat16(), torch.empty_like(keys)
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    append = [_us(lambda: lib.paged_kv_append(None, x, x, keys, other, t, pos, sequences=seq)) for t in (good, bad)]

    S = 70000
    many, short, ones = torch.randn(S, 1, 16, device="cuda", generator=g).bfloat16(), torch.zeros(S, 1, dtype=torch.int32, device="cuda"), torch.ones(S, dtype=torch.int32, device="cuda")
    small = torch.randn(1, 1, 1, 16, device="cuda", generator=g).bfloat16()
    lengths = [_us(lambda: lib.paged_attention(many, small, small, short, lens, 1.0)) for lens in (ones, ones + 1)]
    assert lib.device_error() == 9
    for name, (right, wrong) in (("attention", attend), ("append", append), ("lengths", lengths)):
        assert wrong < 50 * max(right, 20.0), (name, right, wrong)
