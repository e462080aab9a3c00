"""Causal attention over packed prompts and the chunked prefill over the 4-bit cache, against 64-bit forms."""
import math

import numpy as np
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import OjasxB200Error, lib

from q4_plain import attend, gather, random_pool, random_table, rotate, tolerance


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ends(lengths):
    return _ints([0] + list(np.cumsum(lengths)))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _check(q, k, v, lengths, key_lengths, got, scale=None):
    a = e = 0
    for n, m in zip(lengths, key_lengths):
        if n:
            want, big, spread, mass = attend(q[a:a + n], k[e:e + m], v[e:e + m], m - n, scale)
            off, tol = (got[a:a + n].double() - want).abs(), tolerance(q.dtype, want, big, spread, mass, q.shape[-1])
            assert bool((off <= tol).all()), (n, m, float(off.max()), float((off / tol).max()))
        a, e = a + n, e + m


def test_c_entry_refuses_missing_and_unfit_arguments():
    one = 4096
    call = lambda **kw: lib().ojasx_b200_prompt_attention(*{**dict(q=one, qr=128, qh=64, k=one, kr=64, kh=64, v=one, vr=64, vh=64, o=one, e=one, ke=one,
           b=1, n=1, m=1, hq=2, hkv=1, hd=64, sc=-1.0, io=0, ws=one, size=1 << 20, st=None), **kw}.values())  # noqa: E731
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(e=None), dict(ke=None), dict(b=0), dict(n=-1), dict(m=-1), dict(hq=0),
                dict(hkv=0), dict(hq=3, hkv=2), dict(io=2), dict(ws=None), dict(size=100), dict(ws=one + 16), dict(q=one + 8), dict(o=one + 4), dict(kr=66),
                dict(vh=-64), dict(io=1, qh=68)):
        assert call(**bad) == -1, bad
    for bad in (dict(hd=32), dict(hd=256), dict(hq=65)):
        assert call(**bad) == -4, bad
    assert call(n=0) == 0


@pytest.mark.gpu
def test_call_refuses_what_does_not_fit(cuda):
    q, k, e = torch.zeros(4, 4, 64, device=cuda), torch.zeros(4, 2, 64, device=cuda), _ints([0, 4])
    for args in ((q, k, k.bfloat16(), e), (q, k[:3], k[:3], e), (q, k, k, e.long()), (q, k, k, e, _ints([0, 1, 2])), (q[:, :3], k, k, e),
                 (q[..., :32], k[..., :32], k[..., :32], e), (q[0], k, k, e), (q, k, k[:, :1], e)):
        with pytest.raises((ValueError, TypeError)):
            ops.prompt_attention(*args)
    with pytest.raises(TypeError):
        ops.prompt_attention(q.half(), k.half(), k.half(), e)
    with pytest.raises(OjasxB200Error):
        ops.prompt_attention(q.cpu(), k.cpu(), k.cpu(), e.cpu())
    with pytest.raises(ValueError):
        ops.prompt_attention(q, k, k, e, out=torch.zeros(4, 4, 64, device=cuda).bfloat16())
    assert ops.prompt_attention(q[:0], k[:0], k[:0], _ints([0, 0])).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,lengths", [
    (128, 8, 4, [1]), (128, 2, 4, [37]), (64, 1, 1, [1, 2, 31, 32, 33, 63, 64, 65]), (128, 1, 1, [127, 128, 129, 255, 256, 257, 513]),
    (64, 2, 7, [5, 0, 0, 300, 18, 19, 37, 1]), (128, 1, 16, [40, 9]), (64, 1, 64, [7, 70]), (128, 2, 3, [700]), (64, 4, 2, [1] * 70),
    (128, 1, 5, [1030, 3]), (64, 3, 8, [0, 0, 1, 0]), (128, 1, 2, [1500]), (64, 1, 33, [50]), (64, 1, 4, [2100, 40])])
def test_prompts_against_64_bits(cuda, dtype, hd, heads, share, lengths):
    g, n = _gen(sum(lengths) + hd), sum(lengths)
    q, k, v = _randn(g, n, heads * share, hd, dtype=dtype) * 2, _randn(g, n, heads, hd, dtype=dtype), _randn(g, n, heads, hd, dtype=dtype)
    got = ops.prompt_attention(q, k, v, _ends(lengths))
    _check(q, k, v, lengths, lengths, got)
    assert torch.equal(got, ops.prompt_attention(q, k, v, _ends(lengths)))
    _check(q, k, v, lengths, lengths, ops.prompt_attention(q, k, v, _ends(lengths), scale=0.02), 0.02)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,lengths,spread", [(128, [2000], 0), (64, [700, 300], 0), (128, [600], 12)])
def test_fp32_keeps_fp32_accuracy(cuda, hd, lengths, spread):
    """Over all results, errors add up as independent ones do: operands of 22 bits and fp32 sums leave less than 2^-21 of a result (as in
    the test of the decode); twice that is allowed.  `spread`: rows of keys and values that differ by powers of two, up to 2^12."""
    g, n = _gen(30 + hd), sum(lengths)
    q, k, v = _randn(g, n, 4, hd), _randn(g, n, 2, hd), _randn(g, n, 2, hd)
    if spread:
        k = k * torch.exp2(-torch.randint(0, spread, (n, 2, 1), generator=g, device="cuda").float())
        v = v * torch.exp2(-torch.randint(0, spread, (n, 2, 1), generator=g, device="cuda").float())
    got, at, off, size = ops.prompt_attention(q, k, v, _ends(lengths)), 0, 0.0, 0.0
    for m in lengths:
        want = attend(q[at:at + m], k[at:at + m], v[at:at + m], 0)[0]
        off += float((got[at:at + m].double() - want).square().sum())
        size += float(want.square().sum())
        at += m
    assert (off / size) ** 0.5 <= 2.0 ** -20, (off / size) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,lengths,key_lengths", [
    (128, 2, 4, [64], [1000]), (64, 1, 3, [1, 5, 0, 200, 17], [129, 5, 40, 333, 128]), (128, 1, 2, [300, 70, 4], [100, 0, 3]), (64, 2, 1, [1] * 5, [1, 127, 128, 129, 0])])
def test_chunks_behind_and_in_front_of_their_keys(cuda, dtype, hd, heads, share, lengths, key_lengths):
    """More keys than queries (a cached prefix), and fewer: the first queries then see nothing and give zeros."""
    g, n, m = _gen(sum(key_lengths)), sum(lengths), sum(key_lengths)
    q, k, v = _randn(g, n, heads * share, hd, dtype=dtype), _randn(g, m, heads, hd, dtype=dtype), _randn(g, m, heads, hd, dtype=dtype)
    got = ops.prompt_attention(q, k, v, _ends(lengths), _ends(key_lengths))
    _check(q, k, v, lengths, key_lengths, got)
    at = 0
    for a, b in zip(lengths, key_lengths):
        assert not got[at:at + max(0, a - b)].any()
        at += a


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_has_no_part(cuda, dtype, hd, bad):
    """Infinities and NaN in later keys and values, in other sequences and behind the last one."""
    g, lengths = _gen(hd), [150, 300]
    n, rows = sum(lengths), 500
    q, k, v = _randn(g, rows, 4, hd, dtype=dtype), _randn(g, rows, 2, hd, dtype=dtype), _randn(g, rows, 2, hd, dtype=dtype)
    want = ops.prompt_attention(q, k, v, _ends(lengths))
    _check(q, k, v, lengths, lengths, want)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    for t in (k2, v2, q2):
        t[n:] = bad                       # behind the last sequence
    v2[150 + 290:n] = bad                 # seen by the last ten queries of the second sequence alone
    k2[150 + 295:n] = bad
    out = torch.full_like(q, 7)
    assert ops.prompt_attention(q2, k2, v2, _ends(lengths), out=out) is out
    clean = n - 10
    assert torch.isfinite(out[:clean].float()).all()
    _check(q[:clean], k[:clean], v[:clean], [150, 290], [150, 290], out[:clean])
    assert (out[n:] == 7).all()
    assert not torch.isfinite(out[clean:n].float()).any()
    # one value of one dimension: the queries from there on, in that dimension
    v3 = v.clone()
    v3[100, 1, 3] = bad
    out = ops.prompt_attention(q, k, v3, _ends(lengths))[:n].float()
    hit = ~torch.isfinite(out)
    assert hit[100:150, 2:, 3].all() and int(hit.sum()) == 50 * 2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,share", [(64, 1), (128, 1), (128, 4)])
def test_rows_in_front_of_values_that_are_not_finite(cuda, dtype, hd, share):
    """From some token on, every 31st value of a sequence is NaN, in every step of keys that a tile's mask cuts: the rows before that
    token are what they are without, and those from it on are NaN."""
    g = _gen(31)
    lengths = [256] * 24 + [200, 129, 90, 333]
    first = [5 + 17 * b % 80 for b in range(len(lengths))]
    rows = sum(lengths)
    q, k, v = (_randn(g, rows, h, hd, dtype=dtype) for h in (4 * share, 4, 4))
    clean, at = v.clone(), np.cumsum([0] + lengths)
    for a, n, f in zip(at, lengths, first):
        v[a + f:a + n:31] = math.nan
    got = ops.prompt_attention(q, k, v, _ends(lengths))
    for a, n, f in zip(at, lengths, first):
        _check(q[a:a + f], k[a:a + f], clean[a:a + f], [f], [f], got[a:a + f])
        assert torch.isnan(got[a + f:a + n]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,share", [(64, 4, 1), (128, 8, 4)])
def test_every_step_of_short_prompts_counts(cuda, hd, heads, share):
    """Weights are equal and the values of a sequence count its tokens, so that a step of keys whose products a result was read before shows;
    the copies come from memory that the calls in between have pushed out of the cache."""
    lengths = [65 + 7 * b % 130 for b in range(60)]
    rows, at = sum(lengths), np.cumsum([0] + lengths)
    q, k = torch.zeros(rows, heads * share, hd, device=cuda).bfloat16(), torch.zeros(rows, heads, hd, device=cuda).bfloat16()
    place = torch.cat([torch.arange(n, device=cuda) for n in lengths])
    v = (place[:, None, None] // 64).expand(rows, heads, hd).bfloat16().contiguous()       # 0, 1, 2, ...: of the step
    # a row at place p sees p + 1 values whose sums are exact; the rounding to bf16 is off by 2^-8 at most, the reciprocal by far less
    count = (place + 1).double()
    want = torch.stack([(torch.clamp(count - 64 * s, 0, 64) * s) for s in range(4)]).sum(0) / count
    away = torch.empty(64 << 20, dtype=torch.float32, device=cuda)
    for turn in range(20):
        away.fill_(turn)
        got = ops.prompt_attention(q, k, v, _ends(lengths)).double()
        assert bool(((got - want[:, None, None]).abs() <= want[:, None, None] * 2.0 ** -7).all()), turn


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,lengths,key_lengths", [
    (128, 1, 4, [7], [5000]), (128, 2, 4, [100, 33], [2100, 1900]), (64, 3, 3, [40, 1, 0, 130], [2900, 2500, 10, 1500]), (64, 1, 1, [2000], [1999]),
    (128, 2, 8, [600], [600]), (64, 1, 2, [1, 1, 1], [6000, 0, 63]), (128, 1, 64, [3], [2049])])
def test_few_rows_over_many_keys(cuda, dtype, hd, heads, share, lengths, key_lengths):
    """Parts of the rows whose keys several CTAs share; keys behind the last sequence are not finite, and one row's scores end in an outlier."""
    g = _gen(41)
    n, m = sum(lengths), sum(key_lengths)
    q = _randn(g, n + 2, heads * share, hd, dtype=dtype)
    k, v = (_randn(g, m + 70, heads, hd, dtype=dtype) for _ in range(2))
    k[m:], v[m:] = math.nan, math.inf
    k[key_lengths[0] * 3 // 4] *= 6
    got = ops.prompt_attention(q, k, v, _ends(lengths), _ends(key_lengths))
    _check(q, k, v, lengths, key_lengths, got)
    assert torch.equal(got[:n], ops.prompt_attention(q, k, v, _ends(lengths), _ends(key_lengths))[:n])   # joined in one order
    out = torch.full_like(q, 7.0)
    ops.prompt_attention(q, k, v, _ends(lengths), _ends(key_lengths), out=out)
    assert (out[n:] == 7.0).all() and torch.equal(out[:n], got[:n])
    # the values that a row does not see, not finite
    first = lengths[0]
    if first > 1 and key_lengths[0] >= first:
        bad = v.clone()
        bad[key_lengths[0] - 1] = math.nan
        other = ops.prompt_attention(q, k, bad, _ends(lengths), _ends(key_lengths))
        end = key_lengths[0] - 1
        _check(q[:first - 1], k[:end], v[:end], [first - 1], [end], other[:first - 1])
        assert torch.isnan(other[first - 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_short_sequences(cuda, dtype, hd):
    """More parts than the GPU has SMs, of all kinds in turn: without queries, without keys, with values that are not finite behind what
    is seen, with queries that see nothing."""
    g = _gen(hd + 1)
    lengths = [(7 * i) % 41 for i in range(300)] + [300, 0, 257]
    key_lengths = [0 if i % 9 == 4 else n + (i % 5) * 30 if i % 3 else max(0, n - 5) for i, n in enumerate(lengths)]
    n, m = sum(lengths), sum(key_lengths)
    q, k, v = _randn(g, n, 6, hd, dtype=dtype), _randn(g, m, 2, hd, dtype=dtype), _randn(g, m, 2, hd, dtype=dtype)
    want = ops.prompt_attention(q, k, v, _ends(lengths), _ends(key_lengths))
    _check(q, k, v, lengths, key_lengths, want)
    odd, at, e = v.clone(), 0, 0
    keep = torch.ones(n, dtype=torch.bool, device=cuda)
    for i, (a, b) in enumerate(zip(lengths, key_lengths)):
        if i % 4 == 1 and a > 3 and b > 3:      # the last three keys: the last three queries alone see one of them
            odd[e + b - 3:e + b] = math.inf
            keep[at + a - 3:at + a] = False
        at, e = at + a, e + b
    got = ops.prompt_attention(q, k, odd, _ends(lengths), _ends(key_lengths))
    # a part whose values are added one by one adds them in another order: both are within the tolerance of the 64-bit result, and
    # rounded to bf16 (2^-8 of values up to 5)
    bound = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -8 * 5
    assert float((got[keep].float() - want[keep].float()).abs().max()) <= bound
    assert not torch.isfinite(got[~keep].float()).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_and_odd_layouts(cuda, dtype):
    g, n = _gen(3), 90
    x = _randn(g, n, 8 * 64 + 16, dtype=dtype)
    q, k, v = x[:, :256].view(n, 4, 64), x[:, 256:384].view(n, 2, 64), x[:, 384:512].view(n, 2, 64)
    got = ops.prompt_attention(q, k, v, _ends([50, 40]))
    assert torch.equal(got, ops.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), _ends([50, 40])))
    odd = lambda t: torch.cat((t[..., :1], t), -1)[..., 1:]  # noqa: E731
    assert torch.equal(got, ops.prompt_attention(odd(q), odd(k), odd(v), _ends([50, 40])))
    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    assert torch.equal(got, ops.prompt_attention(heads_first(q), heads_first(k), heads_first(v), _ends([50, 40])))
    shared = k[:, :1].expand(n, 2, 64)
    assert torch.equal(ops.prompt_attention(q, shared, shared, _ends([50, 40])), ops.prompt_attention(q, shared.contiguous(), shared.contiguous(), _ends([50, 40])))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_peaked_and_extreme_scores(cuda, dtype):
    g, n = _gen(4), 400
    q, k, v = _randn(g, n, 2, 128, dtype=dtype) * 30, _randn(g, n, 1, 128, dtype=dtype), _randn(g, n, 1, 128, dtype=dtype)
    k[:200] *= 0.01
    k[300] *= 20                      # the largest score comes late
    _check(q, k, v, [n], [n], ops.prompt_attention(q, k, v, _ends([n])))
    q[5, 0, 3] = math.nan
    got = ops.prompt_attention(q, k, v, _ends([n]))
    assert torch.isnan(got[5, 0]).all() and int(torch.isnan(got).sum()) == 128


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_and_streams(cuda, dtype):
    g = _gen(5)
    q, k, v = _randn(g, 300, 8, 128, dtype=dtype), _randn(g, 300, 2, 128, dtype=dtype), _randn(g, 300, 2, 128, dtype=dtype)
    ends = _ends([100, 200])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.prompt_attention(q, k, v, ends)
    for lengths in ([100, 200], [1, 250], [0, 300]):
        q.copy_(_randn(g, 300, 8, 128))
        ends.copy_(_ends(lengths))
        graph.replay()
        _check(q, k, v, lengths, lengths, out)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    want = ops.prompt_attention(q, k, v, ends)
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.prompt_attention(q, k, v, ends))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


# ---------------------------------------------------------------------------------------------- prefill through the cache

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,page,pasts,lengths", [(128, 2, 4, 64, [0], [150]), (64, 2, 3, 16, [100, 0, 7, 33], [40, 5, 0, 130])])
def test_prefill_attends_to_what_the_cache_holds(cuda, dtype, hd, heads, share, page, pasts, lengths):
    g, theta = _gen(6), 1e4
    totals = [p + n for p, n in zip(pasts, lengths)]
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in totals) + 1, page, heads, heads * share, hd, rope_theta=theta)
    random_pool(c, g)
    table, n = random_table(c, totals, g), sum(lengths)
    q, k, v = _randn(g, n, heads * share, hd, dtype=dtype), _randn(g, n, heads, hd, dtype=dtype), _randn(g, n, heads, hd, dtype=dtype)
    got = c.prefill(q, k, v, table, _ints(pasts), _ends(lengths), _ends(totals), sum(totals))
    pool, at = c.unload(), 0
    for b, (p, m) in enumerate(zip(pasts, lengths)):
        if not m:
            continue
        pos = torch.arange(p, p + m, device="cuda")
        turned = rotate(q[at:at + m], pos, theta).to(dtype)      # the three operators in turn: each rounds to the activations' type
        keys, vals = (gather(pool, x, table, b, torch.arange(p + m, device="cuda"), page).to(dtype) for x in ("k", "v"))
        want, big, spread, mass = attend(turned, keys, vals, p)
        # a turned query may be off by a rounding (fp32: 2^-21 of both of a pair; bf16: the other neighbour, 2^-7), which moves the
        # scores by that share of the sum of sizes, the result by twice that times the largest value
        slip = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -20
        tol = tolerance(dtype, want, big, spread, mass, hd) + 2 * big * mass * slip * 2.0 ** -3
        off = (got[at:at + m].double() - want).abs()
        assert bool((off <= tol).all()), (b, float((off / tol).max()))
        at += m


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_prompt_in_chunks_then_tokens(cuda, dtype):
    """A prompt whole and in three chunks leaves the same cache and nearly the same results; decoding the next token with append and
    decode gives what a chunk of one gives."""
    g, n, hd, page = _gen(7), 150, 128, 64
    make = lambda: ops.Q4PagedKVCache(3, page, 2, 8, hd, rope_theta=1e6)  # noqa: E731
    whole, parts, table = make(), make(), _ints([[2, 0, 1]])
    q, k, v = _randn(g, n, 8, hd, dtype=dtype), _randn(g, n, 2, hd, dtype=dtype), _randn(g, n, 2, hd, dtype=dtype)
    m = n - 1
    want = whole.prefill(q[:m], k[:m], v[:m], table, _ints([0]), _ends([m]), _ends([m]), m)
    got, cuts = [], [0, 1, 77, m]
    for a, e in zip(cuts, cuts[1:]):
        got.append(parts.prefill(q[a:e], k[a:e], v[a:e], table, _ints([a]), _ends([e - a]), _ends([e]), e))
    assert torch.equal(whole.pool, parts.pool)
    # the same sums in tiles that begin elsewhere: both are within their tolerance of the 64-bit result, fp32 about 2^-17 of values
    # of size 3 at most, bf16 weights and results half a step (2^-8) each
    bound = 2.0 ** -14 if dtype == torch.float32 else 4 * 2.0 ** -8 * 3
    assert float((torch.cat(got).float() - want.float()).abs().max()) <= bound
    last = slice(m, n)
    one = whole.prefill(q[last], k[last], v[last], table, _ints([m]), _ends([1]), _ends([n]), n)
    turned = parts.append(k[last], v[last], table, _ints([m]), q=q[last])
    step = parts.decode(turned, table, _ints([n]))
    assert torch.equal(whole.pool, parts.pool)
    # decode reads the cache's values in more than bf16: the chunk's keys and values have a rounding of 2^-8 more
    bound = 2.0 ** -14 if dtype == torch.float32 else 0.08
    assert float((step.float() - one.float()).abs().max()) <= bound
