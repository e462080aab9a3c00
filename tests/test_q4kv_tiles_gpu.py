"""Appending packed prompts by whole tiles: enough tokens that the kernel for them runs, whatever GPU it is, with all that the small
cases of the other kernel have.  Also reading more KV heads than a block of the reading kernel has."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import OjasxB200Error

from q4_plain import gather, random_pool, random_table
from test_q4kv_gpu import POOL, THETA, _append_case, _check_append, _ends, _gen, _ints, _randn

pytestmark = pytest.mark.gpu


def _least(hd, heads, q_heads, batch):
    """Tokens from which on tiles are taken: more than 12 units of 1024 values per SM, and 48 per sequence."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    parts = -(-(2 * heads + q_heads) * hd // 1024)
    return (12 * sms + 48 * batch) // parts + 1


def _lengths(lengths, hd, heads, q_heads, tiles=0):
    """The lengths with the one that is None as long as it takes for the tile kernel, and for that many tiles of 16 tokens per SM."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    rest = sum(n or 0 for n in lengths)
    most = max(_least(hd, heads, q_heads, len(lengths)), 16 * tiles * sms) - rest
    return [max(most, 37) if n is None else n for n in lengths]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("theta,queries", [(THETA, True), (None, False)])
@pytest.mark.parametrize("hd,heads,share,page,pasts,lengths,tiles", [
    (128, 2, 4, 64, [5], [None], 0), (64, 3, 3, 16, [0, 5, 16, 31, 8, 100], [17, 0, 1, 50, 8, None], 0), (128, 8, 1, 32, [7] * 40, [1 + 3 * (i % 5) for i in range(39)] + [None], 0),
    (64, 1, 7, 16, [3, 40], [None, 13], 0), (128, 2, 1, 64, [3], [None], 7), (64, 3, 1, 48, [9, 30], [None, 100], 5), (64, 4, 2, 16, [1], [None], 4)])
def test_append_by_tiles(cuda, dtype, theta, queries, hd, heads, share, page, pasts, lengths, tiles):
    """Chunks that begin and end inside pages and tiles, empty ones, rows behind the last sequence; all heads of a tile to a CTA (many
    tiles), some of them, and one."""
    lengths = _lengths(lengths, hd, heads, heads * share if queries else 0, tiles)
    c, before, table, k, v, q = _append_case(hd, heads, share, page, pasts, lengths, dtype, 4, theta, behind=5)
    turned = c.append(k, v, table, _ints(pasts), q=q if queries else None, cu_seqlens=_ends(lengths))
    _check_append(c, before, table, k, v, q, pasts, lengths, turned, theta)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share", [(128, 3, 2), (64, 5, 3)])
def test_one_large_call_is_many_small_ones(cuda, dtype, hd, heads, share):
    """The two kernels give the same codes, scales, minima and queries, bit for bit."""
    g, page = _gen(31), 32
    lengths = _lengths([100, None, 0, 33], hd, heads, heads * share)
    totals = [n + 21 for n in lengths]
    make = lambda: ops.Q4PagedKVCache(sum(-(-n // page) for n in totals), page, heads, heads * share, hd, rope_theta=THETA)  # noqa: E731
    a, b, rows = make(), make(), sum(lengths)
    table = random_table(a, totals, g)
    k, v, q = (_randn(g, rows, n, hd, dtype=dtype) for n in (heads, heads, heads * share))
    whole = a.append(k, v, table, _ints([21] * 4), q=q, cu_seqlens=_ends(lengths))
    starts = np.cumsum([0] + lengths)
    few = _least(hd, heads, heads * share, 4) - 1
    for i, (at, n) in enumerate(zip(starts, lengths)):
        for x in range(0, n, few):
            part = slice(at + x, at + min(n, x + few))
            ends = [0] * (i + 1) + [part.stop - part.start] * (4 - i)
            turned = b.append(k[part], v[part], table, _ints([21 + x if j == i else 0 for j in range(4)]), q=q[part], cu_seqlens=_ints(ends))
            assert torch.equal(turned, whole[part])
    assert torch.equal(a.pool, b.pool)
    a.check()
    b.check()


@pytest.mark.parametrize("hd", [64, 128])
def test_groups_that_are_not_finite_or_of_one_value(cuda, hd):
    n = _least(hd, 1, 0, 1) + 8
    c = ops.Q4PagedKVCache(-(-n // 16), 16, 1, 1, hd)
    x = _randn(_gen(32), n, 1, hd)
    x[3:11] = 0
    x[3] = 3.0
    x[4] = 1.0 / 3
    x[5, 0, :32] = torch.linspace(-1, 1, 32, device=cuda) * 3e38        # a range beyond fp32
    x[6, 0, 5], x[7, 0, 40], x[8, 0, hd - 1] = float("nan"), float("inf"), -float("inf")
    x[9] = torch.linspace(0, 1e-37, hd, device=cuda)
    x[10] = 1000 + torch.linspace(0, 1, hd, device=cuda)
    table = torch.arange(c.num_pages, dtype=torch.int32, device=cuda).view(1, -1)
    c.append(x, x, table, _ints([0]), cu_seqlens=_ends([n]))
    k, v = c.read(table, _ends([n]), n, dtype=torch.float32)
    assert torch.equal(k.nan_to_num(7), v.nan_to_num(7))
    bad = torch.zeros(n, 1, hd // 32, dtype=torch.bool, device=cuda)
    bad[6, 0, 0] = bad[7, 0, 1] = bad[8, 0, -1] = True
    assert torch.equal(torch.isnan(k), bad.repeat_interleave(32, -1))
    scale = c.unload()["k_scales"].transpose(1, 2).reshape(-1, 1, hd // 32)[:n].float().repeat_interleave(32, -1)
    good = ~torch.isnan(k)
    # half a step, and the fp32 rounding of code * scale + minimum (2^-23 of the larger of the two)
    assert bool(((k - x).abs() <= scale * 0.5001 + x.abs() * 2.0 ** -22)[good].all()) and torch.equal(k[3], x[3])


def test_places_that_are_none(cuda):
    """Pages that are none, tokens behind the table and a sequence at a negative position are dropped and reported; all others are kept."""
    g, page, hd = _gen(33), 32, 64
    lengths = _lengths([200, 90, None], hd, 2, 4)
    c = ops.Q4PagedKVCache(sum(-(-(n + 40) // page) for n in lengths), page, 2, 4, hd, rope_theta=THETA)
    before = random_pool(c, g)
    table = random_table(c, [n + 40 for n in lengths], g)
    k, v, q = (_randn(g, sum(lengths), h, hd) for h in (2, 2, 4))
    ends, at = _ends(lengths), [40, 7, 3]
    whole = c.append(k, v, table, _ints(at), q=q, cu_seqlens=ends)
    c.check()
    all_there = c.unload()
    holes = table.clone()
    holes[0, 3], holes[2, 5], holes[2, 6] = -1, c.num_pages, -7
    short = holes[:, :-3].contiguous()         # the longest sequence has no pages for its last tokens
    for tables, starts, kept in ((holes, at, [0, 1, 2]), (short, at, [0, 1, 2]), (holes, [40, -1, 3], [0, 2])):
        c.load(**before)
        turned = c.append(k, v, tables, _ints(starts), q=q, cu_seqlens=ends)
        with pytest.raises(OjasxB200Error):
            c.check()
        after, lost = c.unload(), {int(table[0, 3]), int(table[2, 5]), int(table[2, 6])}
        if tables is short:
            lost |= set(table[2, -3:].tolist())
        for b in range(3):
            pages = [p for p in table[b].tolist() if p >= 0]
            rows = slice(int(ends[b]), int(ends[b + 1]))
            if b in kept:
                assert torch.equal(turned[rows], whole[rows])
            for p in pages:
                want = all_there if b in kept and p not in lost else before
                assert all(torch.equal(after[n][p], want[n][p]) for n in POOL), (b, p)
    c.append(k, v, table, _ints(at), q=q, cu_seqlens=ends)
    c.check()


SCRIPT = r"""
import sys
import torch
sys.path.insert(0, sys.argv[1])
from ojasx_b200 import ops
hd, heads, n = (int(a) for a in sys.argv[2:])
c = ops.Q4PagedKVCache(-(-n // 16), 16, heads, heads, hd)
x, table = torch.ones(n, heads, hd, device="cuda"), torch.arange(c.num_pages, dtype=torch.int32, device="cuda").view(1, -1)
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
pos, mark = ints(0), torch.zeros(1, device="cuda")
got = []
for m in (n, n - 1):
    ends = ints(0, m)
    c.append(x[:m], x[:m], table, pos, cu_seqlens=ends)
    for _ in range(8):
        torch.cuda.synchronize()
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
            mark.erfinv_()
            c.append(x[:m], x[:m], table, pos, cu_seqlens=ends)
            mark.erfinv_()
            torch.cuda.synchronize()
        names = [e.name for e in p.events() if not e.name.startswith("cuda")]
        if sum("erfinv" in s for s in names) == 2:
            got.append(int(any("q4_append_tile_kernel" in s for s in names)))
            break
print(got)
"""


def test_the_tile_kernel_runs_from_there_on(cuda):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", SCRIPT, root, "128", "2", str(_least(128, 2, 0, 1))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
    got = json.loads(run.stdout.strip().splitlines()[-1])
    if len(got) < 2:
        pytest.skip("the profiler records no kernels")
    assert got == [1, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads", [(128, 9), (64, 17)])
def test_read_of_many_heads(cuda, dtype, hd, heads):
    g, starts, lengths = _gen(34), [3, 0, 40], [50, 0, 33]
    c = ops.Q4PagedKVCache(12, 16, heads, heads, hd)
    pool = random_pool(c, g)
    table = random_table(c, [a + n for a, n in zip(starts, lengths)], g)
    k, v = c.read(table, _ends(lengths), sum(lengths), positions=_ints(starts), dtype=dtype)
    for name, got in (("k", k), ("v", v)):
        want = torch.cat([gather(pool, name, table, b, torch.arange(a, a + n, device="cuda"), 16) for b, (a, n) in enumerate(zip(starts, lengths))])
        assert torch.equal(got, want.float().to(dtype)), name
