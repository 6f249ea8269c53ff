"""What a kernel finds in its data on the device (a page outside the pool, a sequence longer than the call
said) is left out and reported, and stops nothing else: waits go on, later steps run, step statuses stay clean."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from test_device_status_gpu import LIMIT, SELFTEST, small_chain  # noqa: E402,F401
from test_kv4_gpu import check_attention, cumulative, filled_cache  # noqa: E402

BF, I32 = torch.bfloat16, torch.int32


def leave_data_error(cuda, code):
    g = torch.Generator(device=cuda).manual_seed(4)
    cache, table, lengths = filled_cache(cuda, [40], 2, 128, 64, g)
    q = torch.randn(1, 16, 128, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [1])
    if code == 0x500:
        ops.kv4_attention(q, cache, torch.full_like(table, cache.shape[0]), lengths, cu, max_new=1, max_len=40)
    else:
        ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=4)


@pytest.mark.parametrize("code", [0x500, 0x502])
def test_waits_do_not_give_up(cuda, code):
    """A wait that has to run its whole bound still does, and its code comes before the data's."""
    assert ops.device_error() == 0
    leave_data_error(cuda, code)
    ops.wait_selftest(LIMIT)
    assert ops.device_error() == SELFTEST
    assert ops.device_error() == code
    assert ops.device_error() == 0


def test_steps_after_it_run_clean(cuda, small_chain):
    chain, args, host, ref = small_chain
    leave_data_error(cuda, 0x500)
    out = chain(*args)
    assert chain.device_status(wait=True) == 0
    assert torch.equal(out.cpu(), ref)
    kept = torch.empty(ref.shape, dtype=BF).pin_memory()
    chain.forward_host(host, kept)
    assert torch.equal(kept, ref)
    g = torch.Generator(device=cuda).manual_seed(5)
    cache, table, lengths = filled_cache(cuda, [3000, 700], 2, 128, 64, g)
    q = torch.randn(2, 16, 128, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [1, 1])
    check_attention(q, cache, table, lengths, cu, ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=3000))
    x = torch.randn(64, 50257, device=cuda, generator=g)
    token, _, _ = ops.sample(x, torch.rand(64, device=cuda, generator=g), temperature=torch.zeros(64, device=cuda))
    assert torch.equal(token, x.argmax(-1))
    assert ops.device_error() == 0x500
    assert ops.device_error() == 0


@pytest.mark.parametrize("lens", [[8192] * 48, [60000, 90, 31]])
def test_rows_of_a_wait_that_ran_out_are_nan(cuda, lens):
    """Under a bound that a copy from memory may pass, a row is right or NaN, and NaN comes with the wait's code.  (The
    bound is looked at every 256 polls: on an idle GPU none runs out and every row is right.)"""
    g = torch.Generator(device=cuda).manual_seed(6)
    cache, table, lengths = filled_cache(cuda, lens, 2, 128, 64, g)
    n = len(lens)
    q = torch.randn(n, 16, 128, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [1] * n)
    flush = torch.empty(1 << 28, dtype=torch.uint8, device=cuda)

    def attend():
        flush.fill_(1)  # the cache is not in L2
        return ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=max(lens))

    want = attend()
    assert ops.device_error() == 0
    limit = ops.get_wait_limit()
    try:
        ops.set_wait_limit(1000)
        for _ in range(10):
            got = attend()
            code = ops.device_error()
            nan = torch.isnan(got.float()).any(2)
            assert torch.equal(got[~nan], want[~nan])
            assert code in (0, 0x510) and bool(nan.any()) <= (code == 0x510)
    finally:
        ops.set_wait_limit(limit)
    assert torch.equal(attend(), want) and ops.device_error() == 0
