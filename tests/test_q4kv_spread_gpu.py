"""Decode over values whose scales differ by powers of two: from token to token, from group to group, and with a token whose scale is
far above all others but whose weight is next to nothing.  Errors are looked at by groups of 32 dimensions, so that a small group next to
a large one counts as much."""
import math

import pytest
import torch

from ojasx_b200 import ops

from q4_plain import attend, gather, random_pool, random_table
from test_q4kv_gpu import _gen, _ints, _randn

pytestmark = pytest.mark.gpu


def _spread(cache, kind, lengths, table, g):
    """A random pool with the scales and minima of its values changed."""
    pool = random_pool(cache, g)
    shape, G = pool["v_scales"].shape, cache.head_dim // 32
    if kind == "tokens":
        by = torch.randint(-14, 15, (*shape[:3], 1), generator=g, device="cuda").float()
    elif kind == "groups":
        by = (torch.arange(G, device="cuda") * (22 // (G - 1)) - 11.0).expand(shape)
    elif kind == "both":
        by = torch.randint(-14, 15, shape, generator=g, device="cuda").float()
    elif kind == "tiny":
        by = torch.full(shape, -60.0, device="cuda")
    else:                # one token of each sequence, its keys far from every query (which are positive here)
        by = torch.zeros(shape, device="cuda")
        for b, n in enumerate(lengths):
            if n:
                at = n // 3
                page, place = int(table[b, at // cache.page_size]), at % cache.page_size
                by[page, :, place] = 22.0 if kind == "outlier" else torch.where(torch.arange(G, device="cuda") == 1, 22.0, 0.0)
                pool["k_codes"][page, :, place] = 0
                pool["k_mins"][page, :, place] = -24.0
    for n in ("v_scales", "v_mins"):
        pool[n] = (pool[n].float() * torch.exp2(by)).to(torch.bfloat16)
    cache.load(**pool)
    return pool


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["tokens", "groups", "both", "tiny", "outlier", "outlier group"])
@pytest.mark.parametrize("hd,heads,share,page,lengths", [(128, 2, 4, 64, [2000, 90]), (64, 2, 7, 16, [1300, 0, 17]), (128, 1, 8, 16, [3])])
def test_decode_of_scales_that_differ(cuda, dtype, kind, hd, heads, share, page, lengths):
    """Per group, errors of independent roundings relative to sum p |v| of the group.  fp32: 2^-20 for operands of 22 bits and fp32
    sums, as where the scales are alike, and the scores' own error: scales that differ leave the result to a few tokens, so that it
    does not average out.  A score is summed in nine fp32 operations at most whose partial results are no larger than `parts`, the sum
    of |q| (|m + 8 s| + |c - 8| s): sqrt(9) * 2^-24 * parts at random, and a result moves by at most twice what its weights do.
    bf16: weights of 11 bits (2^-12 each), sums that the tensor cores keep to 16 bits and the result's half step of 2^-8, which is the
    largest: 2^-8 over all."""
    g = _gen(len(kind) + hd)
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in lengths) + 1, page, heads, heads * share, hd)
    table = random_table(c, lengths, g)
    pool = _spread(c, kind, lengths, table, g)
    q = _randn(g, len(lengths), heads * share, hd, dtype=dtype).abs()
    got = c.decode(q, table, _ints(lengths))
    assert torch.equal(got, c.decode(q, table, _ints(lengths)))
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any()
            continue
        k, v = (gather(pool, x, table, b, torch.arange(n, device="cuda"), page) for x in ("k", "v"))
        want, _, size, _ = attend(q[b:b + 1], k, v, n - 1)
        middle = gather({**pool, "k_codes": torch.full_like(pool["k_codes"], 8)}, "k", table, b, torch.arange(n, device="cuda"), page)
        parts = torch.einsum("hd,mhd->hm", q[b].double(), (middle.abs() + (k - middle).abs()).repeat_interleave(share, 1)).max() * hd ** -0.5
        bound = 2.0 ** -20 + 6 * 2.0 ** -24 * float(parts) if dtype == torch.float32 else 2.0 ** -8
        off, size = ((x.unflatten(-1, (-1, 32)).square().mean((0, 1, 3)).sqrt()) for x in (got[b:b + 1].double() - want, size))
        assert bool((off <= bound * size).all()), (b, (off / size).tolist())
    c.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_of_peaked_scores_and_values_that_are_not_finite(cuda, dtype):
    """Scores that differ by hundreds, queries of zeros, NaN in a query, infinities and NaN in what a query sees, and rising scores."""
    g = _gen(21)
    c = ops.Q4PagedKVCache(8, 64, 1, 4, 128)
    table, n = random_table(c, [500], g), _ints([500])
    pool = random_pool(c, g)
    at = torch.arange(500, device=cuda)
    pool["k_mins"][table[0].long()[at // 64], :, at % 64] = (-4 + at[:, None, None] / 64).to(torch.bfloat16)   # later tokens weigh more and more
    c.load(**pool)
    q = _randn(g, 1, 4, 128, dtype=dtype).abs()
    q[0, 0] *= 30
    q[0, 1] = 0
    k, v = (gather(pool, x, table, 0, at, 64) for x in ("k", "v"))
    want, _, size, _ = attend(q, k, v, 499)
    off, size = ((x[0].unflatten(-1, (-1, 32)).square().mean(-1).sqrt()) for x in (c.decode(q, table, n).double() - want, size))
    # Scores up to 50 are off by 50 * 2^-24 * sqrt(128) at random in fp32, results by twice that (2^-13.9).  In bf16 the tensor cores cut a
    # product of a code at 2^-14 of the largest query value, 3 * 0.17 / sqrt(128) with its scale, 128 of them by 2^-11.6 at most; weights
    # have 2^-12 and results half a step of 2^-8.  The first head's scores and queries are 30 times as large: 2^-6.7.
    assert bool((off[1:] <= (2.0 ** -12 if dtype == torch.float32 else 2.0 ** -7) * size[1:]).all()) and bool((off[0] <= 2.0 ** -6 * size[0]).all())
    q[0, 2, 7] = math.nan
    got = c.decode(q, table, n)
    assert torch.isnan(got[0, 2]).all() and torch.isfinite(got[0, [0, 1, 3]]).all()
    for value in (math.nan, math.inf):
        bad = {name: x.clone() for name, x in pool.items()}
        bad["v_mins"][table[0, 7].long(), 0, 40, 3] = value      # token 488, dimensions 96 to 127
        c.load(**bad)
        got = c.decode(q, table, n)
        assert not torch.isfinite(got[0, [0, 1, 3], 96:]).any() and torch.isfinite(got[0, [0, 1, 3], :96]).all()
        assert torch.isfinite(c.decode(q, table, _ints([488]))[0, [0, 1, 3]]).all()
        bad["k_mins"][table[0, 3].long(), 0, 9, 2] = math.nan
        c.load(**bad)
        assert torch.isnan(c.decode(q, table, n)).all()


def test_scales_with_a_sign_are_refused_or_lose_it(cuda):
    c = ops.Q4PagedKVCache(2, 16, 1, 1, 64)
    pool = random_pool(c, _gen(22))
    for name in ("k_scales", "v_scales"):
        kept = c.pool.clone()
        with pytest.raises(ValueError):
            c.load(**{**pool, name: -pool[name]})
        assert torch.equal(c.pool, kept)
        zero = pool[name].clone()
        zero[0, 0, 3], zero[1, 0, 5, 1] = 0.0, math.nan
        c.load(**{**pool, name: zero})
        kept = c.pool.clone()
        zero[0, 0, 3] = -0.0
        c.load(**{**pool, name: zero})
        assert torch.equal(c.pool, kept) and not bool((c.unload()[name].view(torch.int16) < 0).any())


def test_values_at_the_ends_of_fp32(cuda):
    """The lowest bf16 number is above the lowest fp32 ones: a group with one of those reads as NaN.  Fifteen scales, rounded up, may end
    beyond fp32: the highest reads as infinite.  Up to 3.37e38 everything is finite, and whatever a group holds, the others are kept."""
    c = ops.Q4PagedKVCache(1, 16, 1, 1, 64)
    top = torch.finfo(torch.float32).max
    x = torch.zeros(4, 1, 64, device=cuda)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 5], x[3, 0, 50] = top, -top, -3.38e38, 3.37e38
    c.append(x, x, _ints([[0]]), _ints([0]), cu_seqlens=_ints([0, 4]))
    k, v = c.read(_ints([[0]]), _ints([0, 4]), 4, dtype=torch.float32)
    bad = torch.zeros(4, 1, 64, dtype=torch.bool, device=cuda)
    bad[1, 0, 32:] = True
    scale = c.unload()["k_scales"][0, 0, :4].float()[:, None].repeat_interleave(32, -1)
    for got in (k, v):
        assert torch.equal(torch.isnan(got), bad) and not bool(torch.isfinite(got[0, 0, 3]))
        bad[0, 0, 3] = True
        assert torch.equal(torch.isfinite(got), ~bad)
        # half a step, and the fp32 rounding of code * scale + minimum
        assert bool(((got / 4 - x / 4).abs() <= scale / 4 * 0.5001 + x.abs() / 4 * 2.0 ** -22)[~bad].all())
        bad[0, 0, 3] = False
