"""Attention over prompts at the ends of its range: contexts that take longer than a wait for a phase may."""
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import lib

pytestmark = pytest.mark.gpu


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_a_context_longer_than_a_wait(cuda):
    """24 million keys: a part of the rows takes longer than the eighth of a second after which a wait between the warps of a CTA gives up,
    and its work queue waits as long.  Keys of zeros weigh alike; sums of ones are exact up to 2^24 in steps of one, and beyond it in the
    steps of 64 keys that they are made in (four sums of weights a row, of six million each)."""
    n, m = 300, 24 << 20
    q = torch.ones(n, 64, 64, device=cuda, dtype=torch.bfloat16)
    k = torch.zeros(m, 1, 64, device=cuda, dtype=torch.bfloat16)
    v = torch.ones(m, 1, 64, device=cuda, dtype=torch.bfloat16)
    lib().ojasx_b200_take_device_error()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = ops.prompt_attention(q, k, v, _ints(0, n), _ints(0, m))
    end.record()
    end.synchronize()
    assert lib().ojasx_b200_take_device_error() == 0
    # each of the first rows sees up to 299 keys less, in a step that its mask cuts: sums beyond 2^24 are then off by one part in 2^24
    assert bool(((out.float() - 1).abs() <= 2.0 ** -8).all()), float((out.float() - 1).abs().max())
    print(f"{start.elapsed_time(end):.0f} ms")
