"""Prefill over block tables with entries that are no page: a token without a page weighs nothing, as in a decode."""
import math

import numpy as np
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import OjasxB200Error, lib

from q4_plain import random_pool, random_table, rotate, tolerance, values

THETA = 1e4


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ends(lengths):
    return _ints([0] + list(np.cumsum(lengths)))


def test_c_entries_refuse_marks_on_odd_addresses():
    import ctypes as C
    from ojasx_b200._lib import Q4Cache
    one = 4096
    c = Q4Cache(pool=one, status=one, turns=None, num_pages=1, page_size=16, kv_heads=2, q_heads=4, head_dim=128)
    assert lib().ojasx_b200_q4kv_read_marked(C.addressof(c), one, 1, one, None, one, one, one + 8, 1, 1, 0, None) == -1
    assert lib().ojasx_b200_q4kv_read_marked(C.addressof(c), one, 1, one, None, one, one, one, 0, 1, 0, None) == 0
    assert lib().ojasx_b200_prompt_attention_marked(one, 128, 64, one, 64, 64, one, 64, 64, one, one, one, one + 4, 1, 1, 1, 2, 1, 64, -1.0, 1, None, 0, None) == -1


def _masked(q, k, v, seen):
    """One sequence in 64 bits: q [n, H, hd], k and v [m, Hkv, hd], seen [n, m]; with what `tolerance` asks for."""
    share, hd = q.shape[1] // k.shape[1], q.shape[2]
    kk, vv = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = torch.where(seen, torch.einsum("nhd,mhd->hnm", q.double(), kk) * hd ** -0.5, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out, spread = torch.einsum("hnm,mhd->nhd", p, vv), torch.einsum("hnm,mhd->nhd", p, vv.abs())
    mass = torch.where(seen, torch.einsum("nhd,mhd->hnm", q.double().abs(), kk.abs()) * hd ** -0.5, 0.0).amax(-1).t()[:, :, None]
    return out, vv.abs().max(), spread, mass


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,page,pasts,lengths,holes", [
    (128, 2, 4, 16, [200], [40], [(0, 3), (0, 7), (0, 13)]),                          # in the context and in the chunk
    (64, 2, 3, 16, [100, 0, 7, 33], [40, 5, 0, 130], [(0, 0), (1, 0), (3, 2), (3, 3), (3, 4), (3, 5)]),    # a first page, a whole sequence, four in a row
    (128, 1, 2, 64, [3000], [20], [(0, 0), (0, 1), (0, 40)]),                         # few rows over many keys: shares of the keys, the first without any
    (64, 1, 1, 32, [0], [700], [(0, 0), (0, 1), (0, 10), (0, 21)]),                   # rows that see nothing, and rows whose own tokens are gone
    (128, 4, 2, 64, [64] * 12, [300] * 12, [(b, b % 5) for b in range(12)])])         # more parts than the GPU has SMs
def test_a_token_without_a_page_weighs_nothing(cuda, dtype, hd, heads, share, page, pasts, lengths, holes):
    g = _gen(len(pasts) + hd)
    totals = [p + n for p, n in zip(pasts, lengths)]
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in totals) + 1, page, heads, heads * share, hd, rope_theta=THETA)
    random_pool(c, g)
    table, n = random_table(c, totals, g), sum(lengths)
    for at, (b, p) in enumerate(holes):
        table[b, p] = (-1, c.num_pages)[at % 2]
    q, k, v = (torch.randn(n, h, hd, generator=g, device=cuda).to(dtype) for h in (heads * share, heads, heads))
    call = lambda: c.prefill(q, k, v, table, _ints(pasts), _ends(lengths), _ends(totals), sum(totals))  # noqa: E731
    got = call()
    with pytest.raises(OjasxB200Error):
        c.check()
    assert torch.equal(got, call())
    pool, at = c.unload(), 0
    for b, (past, m) in enumerate(zip(pasts, lengths)):
        if not m:
            continue
        tokens = torch.arange(past + m, device=cuda)
        ids = table[b].long()[tokens // page]
        there = (ids >= 0) & (ids < c.num_pages)
        keys, vals = (values(*(pool[x + part][ids.clamp(0, c.num_pages - 1), :, tokens % page] for part in ("_codes", "_scales", "_mins"))).to(dtype).double() for x in "kv")
        turned = rotate(q[at:at + m], torch.arange(past, past + m, device=cuda), THETA).to(dtype)
        seen = there & (tokens <= past + torch.arange(m, device=cuda)[:, None])
        want, big, spread, mass = _masked(turned, keys, vals, seen)
        # (a turned query may be off by a rounding: as in the test of the prefill without holes)
        slip = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -20
        tol = tolerance(dtype, want, big, spread, mass, hd) + 2 * big * mass * slip * 2.0 ** -3
        off = (got[at:at + m].double() - want).abs()
        assert bool((off <= tol).all()), (b, float((off / tol).max()))
        assert not got[at:at + m][~seen.any(1)].any()
        at += m


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_chunk_of_one_is_a_step(cuda, dtype):
    """Over a table with holes, append and decode give what a chunk of one token gives: both are within their tolerance of the same sum,
    and the chunk's keys and values have a rounding to the activations' type more (as where no page is missing)."""
    g, n, hd = _gen(9), 500, 128
    c = ops.Q4PagedKVCache(40, 16, 2, 8, hd, rope_theta=THETA)
    random_pool(c, g)
    table = random_table(c, [n + 1], g)
    table[0, 2], table[0, 9], table[0, 30] = -1, 99, -1
    q, k, v = (torch.randn(1, h, hd, generator=g, device=cuda).to(dtype) for h in (8, 2, 2))
    one = c.prefill(q, k, v, table, _ints([n]), _ends([1]), _ends([n + 1]), n + 1)
    step = c.decode(c.append(k, v, table, _ints([n]), q=q), table, _ints([n + 1]))
    assert float((step.float() - one.float()).abs().max()) <= (2.0 ** -14 if dtype == torch.float32 else 0.08)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [48, 80, 144, 1008])
def test_pages_of_any_multiple_of_a_tile(cuda, dtype, page):
    """The same tokens in pages of 16 and of other sizes: the same codes and the same bits from every call."""
    g, hd, pasts, lengths = _gen(page), 64, [0, 37, 1000], [300, 1, 77]
    totals = [p + n for p, n in zip(pasts, lengths)]
    n, m = sum(lengths), sum(totals)
    k, v, q = (torch.randn(m, h, hd, generator=g, device=cuda).to(dtype) for h in (2, 2, 6))
    got = []
    for size in (16, page):
        c = ops.Q4PagedKVCache(sum(-(-t // size) for t in totals) + 2, size, 2, 6, hd, rope_theta=THETA)
        table = random_table(c, totals, g)
        first = torch.cat([torch.arange(e - t, e - t + p) for e, t, p in zip(np.cumsum(totals), totals, pasts)]).to(cuda)
        then = torch.cat([torch.arange(e - t + p, e) for e, t, p in zip(np.cumsum(totals), totals, pasts)]).to(cuda)
        c.append(k[first], v[first], table, _ints([0] * 3), cu_seqlens=_ends(pasts))
        out = c.prefill(q[then], k[then], v[then], table, _ints(pasts), _ends(lengths), _ends(totals), m)
        got.append((out, c.decode(q[:3], table, _ints(totals)), *c.read(table, _ends(totals), m, dtype=dtype)))
        c.check()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_captured_prefill_follows_tables_and_positions(cuda, dtype):
    """One graph for chunks of up to 64 tokens over up to 400 cached ones; replayed on two streams in turn, with holes the second time."""
    g, hd, most = _gen(13), 128, 400
    c = ops.Q4PagedKVCache(60, 16, 2, 8, hd, rope_theta=THETA)
    random_pool(c, g)
    q, k, v = (torch.randn(64, h, hd, generator=g, device=cuda).to(dtype) for h in (8, 2, 2))
    tables, pos, ends, totals = random_table(c, [200, 200], g, width=13), _ints([0, 0]), _ends([10, 20]), _ends([10, 20])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = c.prefill(q, k, v, tables, pos, ends, totals, most)
    for turn, (pasts, lengths) in enumerate((([100, 0], [30, 34]), ([3, 150], [1, 50]), ([136, 136], [64, 0]))):
        now = random_table(c, [200, 200], g, width=13)
        if turn == 1:
            now[1, 4] = now[0, 0] = -1
        tables.copy_(now)
        pos.copy_(_ints(pasts))
        ends.copy_(_ends(lengths))
        totals.copy_(_ends([p + n for p, n in zip(pasts, lengths)]))
        kept = c.pool.clone()
        with torch.cuda.stream(torch.cuda.current_stream() if turn % 2 else side):
            side.wait_stream(torch.cuda.default_stream())
            graph.replay()
        torch.cuda.synchronize()
        pool = c.pool.clone()
        c.pool.copy_(kept)
        want = c.prefill(q, k, v, now, _ints(pasts), _ends(lengths), _ends([p + n for p, n in zip(pasts, lengths)]), sum(pasts) + sum(lengths))
        rows = sum(lengths)
        assert torch.equal(c.pool, pool)
        # the plan of the captured call is for 400 keys: sums may be shared out differently
        bound = 2.0 ** -15 if dtype == torch.float32 else 2.0 ** -6
        assert float((out[:rows].float() - want[:rows].float()).abs().max()) <= bound * float(want[:rows].float().abs().max())
