"""Attention over prompts at the ends of its range: contexts that take longer than a wait for a phase may."""
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import lib

from q4_plain import tolerance
from test_prefill_holes_gpu import _masked as masked

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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,n,m", [(64, 150, 150), (128, 40, 3000)])
def test_a_key_with_an_infinity(cuda, dtype, hd, n, m):
    """A score of -inf weighs nothing, one of +inf or NaN leaves no result: by the sign of the one element of a query that meets it."""
    g = torch.Generator(device="cuda").manual_seed(hd)
    q, k, v = (torch.randn(r, h, hd, generator=g, device=cuda).to(dtype) for r, h in ((n, 4), (m, 2), (m, 2)))
    at, first = m - n // 2, n - n // 2          # the key, and the first query that sees it
    k[at, 0, 5] = -float("inf")                 # (of the first KV head, which two query heads share)
    q[:, :2, 5] = q[:, :2, 5].abs().clamp(min=0.25)
    q[first + 3, 0, 5] *= -1
    q[first + 4, 1, 5] = 0
    got = ops.prompt_attention(q, k, v, _ints(0, n), _ints(0, m)).double()
    finite = torch.ones(n, 4, dtype=torch.bool, device=cuda)
    finite[first + 3, 0] = finite[first + 4, 1] = False
    assert torch.equal(torch.isfinite(got).all(-1), finite) and not torch.isfinite(got[~finite]).any()
    keys = k.clone()
    keys[at, 0] = 0
    seen = torch.arange(m, device=cuda) <= torch.arange(m - n, m, device=cuda)[:, None]
    for heads, see in ((slice(0, 2), seen & (torch.arange(m, device=cuda) != at)), (slice(2, 4), seen)):
        kv = slice(heads.start // 2, heads.start // 2 + 1)
        want, big, spread, mass = masked(q[:, heads], keys[:, kv].double(), v[:, kv].double(), see)
        tol = tolerance(dtype, want, big, spread, mass, hd)
        assert bool(((got[:, heads] - want).abs() <= tol)[finite[:, heads]].all())


@pytest.mark.parametrize("power", [-120, -45, -37, 0, 60, 95])
@pytest.mark.parametrize("what", ["keys", "values", "one dimension"])
def test_fp32_operands_of_any_size(cuda, what, power):
    """Keys of any size against queries that bring the scores back; values of any size up to 2^100, with errors of 2^-59 where they are small;
    one dimension of all rows far above or below the others.  Relative errors are independent ones as in the tests of fp32 accuracy, 2^-20;
    what is more than 2^-17 below its row's largest is off by 2^-40 of that at most, and so is a mean of such values.  The exponent of a
    row of values is added to its scores (up to 16 here, in powers of two), whose sum fp32 rounds to 2^-24 of its size, power + 16; a
    weight moves by ln 2 of that, and a result by twice what its weights do."""
    if what == "one dimension" and abs(power) > 60:
        power //= 4
    g = torch.Generator(device="cuda").manual_seed(7)
    n = 400
    q, k, v = (torch.randn(n, h, 64, generator=g, device=cuda) for h in (4, 2, 2))
    if what == "keys":
        k, q = k * 2.0 ** power, q * 2.0 ** -power
    elif what == "values":
        v = v * 2.0 ** power
    else:
        v[..., 9] *= 2.0 ** power
    got = ops.prompt_attention(q, k, v, _ints(0, n)).double()
    seen = torch.arange(n, device=cuda) <= torch.arange(n, device=cuda)[:, None]
    want, _, _, _ = masked(q, k.double(), v.double(), seen)
    most = float(v.abs().max())
    floor = max(2.0 ** -59, 2.0 ** -40 * most)
    for part in ((slice(9), slice(10, 64)), (slice(9, 10),)):
        off, size = (torch.cat([x[..., s] for s in part], -1).square().mean().sqrt() for x in (got - want, want))
        weights = 2 * 0.7 * 2.0 ** -24 * (abs(power) + 16) if what == "values" else 0.0
        assert float(off) <= (2.0 ** -20 + weights) * float(size) + floor, (float(off), float(size))
