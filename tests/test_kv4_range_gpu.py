"""The 4-bit cache's attention over the rest of its range: batches of several launches, values of any size, rows
and pages that the host cannot see to be missing.  Plain forms and their tolerances: test_kv4_gpu.py."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from test_kv4_gpu import check_attention, cumulative, filled_cache  # noqa: E402

BF, F64, I32 = torch.bfloat16, torch.float64, torch.int32


# ------------------------------------------------------------------------------------------------
# more sequences than one launch takes (1024)
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seqs", [1024, 1025, 1043, 2050])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (24, 24, 64)])
@pytest.mark.parametrize("longest", [1000, 8192])  # of a launch that cuts no segment, and of one that may
def test_many_sequences(cuda, seqs, hq, hkv, d, longest):
    """The last launch holds a few sequences only: it keeps the plan of the first, with or without a workspace."""
    g = torch.Generator(device=cuda).manual_seed(seqs + d)
    lens = [(7 * b) % 41 for b in range(seqs)]
    lens[3], lens[-1] = 150, 150
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, 32, g, fill=0xFF)
    new = [min(1, n) for n in lens]
    q = torch.randn(sum(new), hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    wide = torch.full((seqs, -(-longest // 32)), -1, dtype=I32, device=cuda)  # room for `longest` tokens a sequence
    wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
    out = ops.kv4_attention(q, cache, wide, lengths, cu, max_new=1, max_len=longest)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    some = [b for b in range(seqs) if lens[b] and (b < 40 or b % 37 == 0 or b > 1000)]
    rows = cu[:-1][some].long()
    check_attention(q[rows], cache, table[some], lengths[some], cumulative(cuda, [1] * len(some)), out[rows])
