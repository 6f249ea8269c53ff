"""B200TextDecoder beyond plain prompts: rows that cannot be drawn from, prompts with positions and features of their
own.  Plain forms and their tolerance: test_decoder_gpu.py."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from rldx_b200.decoder import B200TextDecoder  # noqa: E402
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


@torch.no_grad()
def test_generate_with_positions(cuda):
    """The same tokens where the tables hold the same rows elsewhere, and those of single steps with the same positions."""
    stack, embed, head, cos, sin, dec = make(cuda)
    prompts = [[1, 5, 9, 200, 31], list(range(40, 140))]
    u = torch.rand(8, 2, generator=torch.Generator().manual_seed(2))
    want = dec.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95)
    moved = B200TextDecoder(stack.layers, stack.norm, embed, head, *(torch.cat([torch.full_like(t[:50], 7.0), t]) for t in (cos, sin)),
                            device=cuda)
    at = [torch.arange(len(p)) + 50 for p in prompts]
    assert moved.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95, positions=at) == want
    assert moved.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95) != want
    # as vision tokens stand: several in one place, the text after them one past the largest
    rows = dec.embed[torch.tensor(prompts[1][:40], device=cuda)]
    place = torch.cat([torch.arange(10), 10 + torch.arange(20) // 5 % 4, torch.arange(14, 24)])
    got = dec.generate([rows], 6, u=u[:6, :1], temperature=0.0, positions=[place])[0]
    cache, hidden, new, pos, ids = dec.new_cache(1, 60), rows, [40], place, []
    for i in range(6):
        ids.append(int(dec.forward(hidden, cache, new, pos).float().argmax()))
        hidden, new, pos = dec.embed[ids[-1]][None], [1], torch.tensor([24 + i])
    assert got == ids
    assert ops.device_error() == 0
