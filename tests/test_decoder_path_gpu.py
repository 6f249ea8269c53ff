"""B200TextDecoder beyond plain prompts: rows that cannot be drawn from, prompts with positions and features of their
own.  Plain forms and their tolerance: test_decoder_gpu.py."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from test_decoder_gpu import make  # noqa: E402


@torch.no_grad()
def test_a_sequence_of_nan_is_reported(cuda):
    dec = make(cuda)[-1]
    bad = dec.embed[:6].clone()
    bad[3] = float("nan")
    u = torch.rand(4, 2, generator=torch.Generator().manual_seed(1))
    with pytest.raises(RuntimeError, match="sequence 1 has no logit that is a number at its token 0"):
        dec.generate([[1, 2, 3], bad], 4, u=u)
    assert ops.device_error() == 0
    assert len(dec.generate([[1, 2, 3], bad[:3]], 4, u=u)[1]) == 4
