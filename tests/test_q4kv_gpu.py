"""The 4-bit paged KV cache: its format bit for bit, the rotation on the way in, reading back, and attention of single tokens
against plain 64-bit forms, at the places where pages, tiles and sequences end."""
import numpy as np
import pytest
import torch

from ojasx_b200 import ops
from ojasx_b200._lib import OjasxB200Error, Q4Cache, lib

from q4_plain import attend, gather, quantize, random_pool, random_table, rotate, tolerance, values

THETA = 1e6
POOL = [n + p for n in ("k", "v") for p in ("_codes", "_scales", "_mins")]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _ends(lengths):
    return _ints([0] + list(np.cumsum(lengths)))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


# ---------------------------------------------------------------------------------------------- refusals (no GPU)

def test_c_entries_refuse_missing_and_unfit_arguments():
    import ctypes as C
    L = lib()
    one = 4096   # an address that no call gets as far as using
    kept = []

    def cache(**kw):
        c = Q4Cache(**{**dict(pool=one, status=one, turns=None, num_pages=1, page_size=16, kv_heads=2, q_heads=4, head_dim=128), **kw})
        kept.append(c)
        return C.addressof(c)

    bad_caches = [(None, -1)] + [(cache(**kw), -1) for kw in (dict(pool=None), dict(status=None), dict(num_pages=0), dict(kv_heads=0), dict(q_heads=3),
                                 dict(q_heads=0), dict(pool=one + 8))]
    bad_caches += [(cache(**kw), -4) for kw in (dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(head_dim=96), dict(head_dim=0))]
    good = cache()
    append = lambda **kw: L.ojasx_b200_q4kv_append(*{**dict(c=good, k=one, ks=128, v=one, vs=128, q=None, qs=0, qo=None, table=one, mp=1, pos=one,
             ends=None, n=1, b=1, io=0, st=None), **kw}.values())  # noqa: E731
    decode = lambda **kw: L.ojasx_b200_q4kv_decode(*{**dict(c=good, q=one, o=one, table=one, mp=1, n=one, b=1, sc=-1.0, io=1, ws=one, size=1 << 30,
             st=None), **kw}.values())  # noqa: E731
    read = lambda **kw: L.ojasx_b200_q4kv_read(*{**dict(c=good, table=one, mp=1, ends=one, pos=None, k=one, v=one, n=1, b=1, io=0, st=None),
                                               **kw}.values())  # noqa: E731
    for call in (append, decode, read):
        for c, code in bad_caches:
            assert call(c=c) == code
        for bad in (dict(table=None), dict(mp=0), dict(b=0), dict(io=7)):
            assert call(**bad) == -1, bad
        assert call(c=cache(page_size=4096), mp=1 << 20) == -5
    for bad in (dict(k=None), dict(v=None), dict(pos=None), dict(n=2), dict(n=-1), dict(k=one + 4), dict(ks=2), dict(q=one), dict(q=one, qo=one + 8)):
        assert append(**bad) == -1, bad
    assert append(n=0, ends=one) == 0
    for bad in (dict(q=None), dict(o=None), dict(n=None), dict(q=one + 2), dict(o=one + 8), dict(ws=None), dict(size=1000), dict(ws=one + 4)):
        assert decode(**bad) == -1, bad
    for bad in (dict(ends=None), dict(k=None), dict(v=one + 1), dict(n=-1)):
        assert read(**bad) == -1, bad
    assert read(n=0) == 0
    assert L.ojasx_b200_q4kv_page_bytes(8, 64, 128) == 8 * 64 * 160 and L.ojasx_b200_q4kv_page_bytes(1, 16, 64) == 16 * 80
    assert L.ojasx_b200_q4kv_page_bytes(8, 20, 128) == 0 and L.ojasx_b200_q4kv_page_bytes(8, 64, 32) == 0


def test_cache_refuses_unfit_geometry():
    for bad in (dict(num_pages=0), dict(page_size=8), dict(page_size=24), dict(kv_heads=3), dict(head_dim=96), dict(rope_theta=0.0)):
        with pytest.raises(ValueError):
            ops.Q4PagedKVCache(**{**dict(num_pages=4, page_size=16, kv_heads=2, q_heads=4, head_dim=64), **bad}, device="cuda:0")


@pytest.mark.gpu
def test_calls_refuse_what_does_not_fit(cuda):
    c = ops.Q4PagedKVCache(4, 16, 2, 4, 64)
    t, p = _ints([[0, 1]]), _ints([0])
    k, q = torch.zeros(1, 2, 64, device=cuda), torch.zeros(1, 4, 64, device=cuda)
    for args, kw in (((k, k.bfloat16(), t, p), {}), ((k[:, :1], k, t, p), {}), ((k, k, t.long(), p), {}), ((k, k, t, _ints([0, 0])), {}),
                     ((k, k, t[0], p), {}), ((k, k, t, p), dict(q=q[:, :3])), ((torch.cat((k, k)), torch.cat((k, k)), t, p), {}),
                     ((k, k, t, p), dict(cu_seqlens=_ints([0]))), ((k, k, _ints([[0, 9, 1, 9]])[:, ::2], p), {})):
        with pytest.raises((ValueError, TypeError)):
            c.append(*args, **kw)
    with pytest.raises(TypeError):
        c.append(k.half(), k.half(), t, p)
    with pytest.raises(OjasxB200Error):
        c.append(k.cpu(), k.cpu(), t, p)
    for bad in (q[:, :2], torch.cat((q, q))):
        with pytest.raises(ValueError):
            c.decode(bad, t, p)
    with pytest.raises(ValueError):
        c.decode(q, t, p, out=torch.zeros(1, 4, 64, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        c.load(**{n: torch.zeros(1, device=cuda) for n in POOL})


# ---------------------------------------------------------------------------------------------- format

@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,page", [(64, 3, 16), (128, 2, 48)])
def test_load_and_unload_are_inverse(cuda, hd, heads, page):
    c = ops.Q4PagedKVCache(3, page, heads, heads, hd)
    pool = random_pool(c, _gen(hd))
    back = c.unload()
    for n in POOL:
        assert torch.equal(back[n], pool[n]), n


def _append_case(hd, heads, share, page, pasts, lengths, dtype, seed, theta=THETA, spare=2, behind=0):
    g = _gen(seed)
    totals = [p + n for p, n in zip(pasts, lengths)]
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in totals) + spare, page, heads, heads * share, hd, rope_theta=theta)
    before = random_pool(c, g)
    table = random_table(c, totals, g)
    rows = sum(lengths) + behind
    k, v, q = _randn(g, rows, heads, hd, dtype=dtype), _randn(g, rows, heads, hd, dtype=dtype), _randn(g, rows, heads * share, hd, dtype=dtype)
    return c, before, table, k, v, q


def _check_append(c, before, table, k, v, q, pasts, lengths, turned, theta):
    """Values of V bit for bit, keys within half a step and the rotation's rounding, everything else in the pool as it was."""
    after, page = c.unload(), c.page_size
    pos = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(pasts, lengths)])
    seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(lengths)]).long()
    n, ids, at = pos.numel(), table[seq, pos // page].long(), pos % page
    for part, want in zip(("_codes", "_scales", "_mins"), quantize(v[:n])):
        assert torch.equal(after["v" + part][ids, :, at], want), "v" + part
    want = rotate(k[:n], pos, theta) if theta else k[:n].double()
    # rotation: the fraction of a turn is rounded to fp32 (2^-26 turns), cos and sin to 2 steps, products and sum to 3 half steps
    half = c.head_dim // 2
    size = (k[:n, :, :half].double().abs() + k[:n, :, half:].double().abs()).repeat(1, 1, 2) * 2.0 ** -21
    codes, scales, mins = (after["k" + part][ids, :, at] for part in ("_codes", "_scales", "_mins"))
    step = scales.double().repeat_interleave(32, -1)
    off = (values(codes, scales, mins) - want).abs()
    assert bool((off <= step * (0.5 + 2.0 ** -15) + size).all()), float((off / step).max())
    grp, slack = want.unflatten(-1, (-1, 32)), size.unflatten(-1, (-1, 32)).amax(-1)
    lo, hi = grp.amin(-1), grp.amax(-1)
    assert bool((mins.double() <= lo + slack).all()) and bool((mins.double() >= lo - slack - lo.abs() * 2.0 ** -7).all())
    # one step of bf16 up at most (2^-7), from a range that is off by both ends' rounding
    assert bool((scales.double() <= ((hi - mins.double() + 2 * slack) / 15) * (1 + 2.0 ** -7)).all())
    if theta == 0 or theta is None:
        for part, exact in zip(("_codes", "_scales", "_mins"), quantize(k[:n])):
            assert torch.equal(after["k" + part][ids, :, at], exact), "k" + part
    for name in POOL:
        kept, now = before[name].clone(), after[name].clone()
        kept[ids, :, at], now[ids, :, at] = 0, 0
        assert torch.equal(kept, now), name
    if turned is not None:
        qw = rotate(q[:n], pos, theta) if theta else q[:n].double()
        size = (q[:n, :, :half].double().abs() + q[:n, :, half:].double().abs()).repeat(1, 1, 2) * 2.0 ** -21
        if q.dtype == torch.bfloat16:
            size = size + qw.abs() * 2.0 ** -8
        assert bool(((turned[:n].double() - qw).abs() <= size).all())
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,page,pasts", [(128, 8, 4, 64, [1000]), (128, 1, 1, 16, [0, 1, 15, 16, 17, 31]), (64, 2, 7, 32, [0, 63, 64, 1 << 20]),
                                                       (128, 3, 16, 128, [127, 128, 5])])
def test_append_single_tokens(cuda, dtype, hd, heads, share, page, pasts):
    real = [min(p, 4000) for p in pasts]     # (a far position needs its page only)
    lengths = [1] * len(pasts)
    c, before, table, k, v, q = _append_case(hd, heads, share, page, real, lengths, dtype, 3)
    if real != pasts:
        wide = torch.full((len(pasts), max(pasts) // page + 1), -1, dtype=torch.int32, device="cuda")
        for b, p in enumerate(pasts):
            wide[b, p // page] = table[b, real[b] // page]
        table = wide
    turned = c.append(k, v, table, _ints(pasts), q=q)
    _check_append(c, before, table, k, v, q, pasts, lengths, turned, THETA)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("theta", [THETA, None])
@pytest.mark.parametrize("hd,heads,share,page,pasts,lengths", [(128, 2, 4, 64, [0], [200]), (64, 3, 3, 16, [0, 5, 16, 31, 8, 100], [17, 0, 1, 50, 8, 3]),
                                                               (128, 8, 1, 32, [7] * 40, [1 + 3 * (i % 5) for i in range(40)])])
def test_append_packed(cuda, dtype, theta, hd, heads, share, page, pasts, lengths):
    """Chunks that begin and end inside pages and tiles, empty ones, rows behind the last sequence."""
    c, before, table, k, v, q = _append_case(hd, heads, share, page, pasts, lengths, dtype, 4, theta, behind=5)
    turned = c.append(k, v, table, _ints(pasts), q=q, cu_seqlens=_ends(lengths))
    _check_append(c, before, table, k, v, q, pasts, lengths, turned, theta)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_append_views_of_a_fused_projection(cuda, packed):
    """q, k and v as column ranges of one tensor are taken where they lie; odd ones are copied."""
    g, B = _gen(5), 5
    c = ops.Q4PagedKVCache(B, 16, 2, 6, 64, rope_theta=THETA)
    before = random_pool(c, g)
    table, ends = random_table(c, [1] * B, g), _ends([1] * B) if packed else None
    x = _randn(g, B, 10 * 64 + 8, dtype=torch.bfloat16)
    q, k, v = x[:, :384].view(B, 6, 64), x[:, 384:512].view(B, 2, 64), x[:, 512:640].view(B, 2, 64)
    turned = c.append(k, v, table, _ints([0] * B), q=q, cu_seqlens=ends)
    _check_append(c, before, table, k, v, q, [0] * B, [1] * B, turned, THETA)
    odd = _randn(g, B, 2, 65, dtype=torch.bfloat16)[:, :, 1:]     # heads 65 apart, at odd addresses
    first = c.unload()
    c.append(odd, odd, table, _ints([0] * B), cu_seqlens=ends)
    _check_append(c, first, table, odd, odd, None, [0] * B, [1] * B, None, THETA)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_groups_of_one_value_of_wide_range_and_not_finite(cuda, packed):
    c = ops.Q4PagedKVCache(1, 16, 1, 1, 128)
    x = torch.zeros(8, 1, 128, device=cuda)
    x[0] = 3.0
    x[1] = 1.0 / 3
    x[2, 0, :64] = torch.linspace(-1, 1, 64, device=cuda) * 3e38
    x[2, 0, 96:] = torch.linspace(-1, 1, 32, device=cuda) * 3e38      # a range beyond fp32
    x[3, 0, 5] = float("nan")
    x[4, 0, 40] = float("inf")
    x[5, 0, 70] = -float("inf")
    x[6] = torch.linspace(0, 1e-37, 128, device=cuda)
    x[7] = 1000 + torch.linspace(0, 1, 128, device=cuda)
    table, pos, ends = _ints([[0]]), _ints([0]), _ends([8])
    if packed:
        c.append(x, x, table, pos, cu_seqlens=ends)
    else:
        for i in range(8):
            c.append(x[i:i + 1], x[i:i + 1], table, _ints([i]))
    k, v = c.read(table, ends, 8, dtype=torch.float32)
    assert torch.equal(k.nan_to_num(7), v.nan_to_num(7))
    bad = torch.zeros(8, 1, 4, dtype=torch.bool, device=cuda)
    bad[3, 0, 0] = bad[4, 0, 1] = bad[5, 0, 2] = True
    assert torch.equal(torch.isnan(k), bad.repeat_interleave(32, -1))
    good = ~torch.isnan(k)
    scale = c.unload()["k_scales"][0, 0, :8].float()[:, None].repeat_interleave(32, -1)
    # half a step, and the fp32 rounding of code * scale + minimum (2^-23 of the larger of the two)
    assert bool(((k - x).abs() <= scale * 0.5001 + x.abs() * 2.0 ** -22)[good].all())
    assert torch.equal(k[0], x[0])     # a value that bf16 holds is kept as it is


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_tokens_without_a_page_are_dropped_and_reported(cuda, packed):
    g = _gen(6)
    c = ops.Q4PagedKVCache(4, 16, 2, 2, 64)
    before = random_pool(c, g)
    k = _randn(g, 5, 2, 64)
    table, ends = _ints([[0], [-1], [4], [2], [1]]), _ends([1] * 5) if packed else None
    c.append(k, k, table, _ints([3, 3, 3, 16, 9]), cu_seqlens=ends)      # page -1, page 4 of 4, a position behind the table
    after = c.unload()
    for name in POOL:
        kept, now = before[name].clone(), after[name].clone()
        for page, at in ((0, 3), (1, 9)):
            assert page or not torch.equal(kept[page, :, at], now[page, :, at]) or name.endswith("scales") or name.endswith("mins")
            kept[page, :, at], now[page, :, at] = 0, 0
        assert torch.equal(kept, now), name
    with pytest.raises(OjasxB200Error):
        c.check()
    c.check()
    kk, vv = c.read(table, _ends([1, 1, 1, 0, 0]), 3, dtype=torch.float32)
    assert not kk[1:].any() and not vv[1:].any() and kk[0].any()
    with pytest.raises(OjasxB200Error):
        c.check()
    # a decode passes over them: a sequence whose second page is none has the first one's tokens
    q = _randn(g, 1, 2, 64)
    got, want = c.decode(q, _ints([[0, -1]]), _ints([30])), c.decode(q, _ints([[0]]), _ints([16]))
    assert torch.allclose(got, want, rtol=2.0 ** -20, atol=0)
    with pytest.raises(OjasxB200Error):
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 40])   # of a sequence: either kernel
def test_a_negative_position_is_no_place(cuda, tokens):
    g = _gen(11)
    c = ops.Q4PagedKVCache(6, 32, 2, 4, 64, rope_theta=THETA)
    table, ends = _ints([[0, 1], [2, 3]]), _ends([tokens, tokens])
    k, v, q = _randn(g, 2 * tokens, 2, 64), _randn(g, 2 * tokens, 2, 64), _randn(g, 2 * tokens, 4, 64)
    whole, before = c.append(k, v, table, _ints([0, 5]), q=q, cu_seqlens=ends), c.pool.clone()
    c.check()
    c.pool.zero_()
    turned = c.append(k, v, table, _ints([-1, 5]), q=q, cu_seqlens=ends)
    with pytest.raises(OjasxB200Error):
        c.check()
    assert not c.pool[:2].any() and torch.equal(c.pool[2:], before[2:]) and torch.equal(turned[tokens:], whole[tokens:])
    c.read(table, ends, 2 * tokens, positions=_ints([0, -4]))
    with pytest.raises(OjasxB200Error):
        c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_length_beyond_the_table_is_reported(cuda, dtype):
    g = _gen(12)
    c = ops.Q4PagedKVCache(6, 32, 2, 4, 64)
    pool = random_pool(c, g)
    table, q = random_table(c, [64, 50], g), _randn(g, 2, 4, 64, dtype=dtype)
    _check_decode(c, pool, table, [64, 50], q, c.decode(q, table, _ints([64, 50])))
    c.check()
    got = c.decode(q, table, _ints([65, 50]))
    with pytest.raises(OjasxB200Error):
        c.check()
    _check_decode(c, pool, table, [64, 50], q, got)   # the tokens that there is room for
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,page,starts,lengths", [(128, 2, 64, [0], [130]), (64, 3, 16, [3, 0, 16, 40], [5, 0, 33, 1])])
def test_read_gives_the_values(cuda, dtype, hd, heads, page, starts, lengths):
    g = _gen(7)
    c = ops.Q4PagedKVCache(12, page, heads, heads, hd)
    pool, rows = random_pool(c, g), sum(lengths)
    table = random_table(c, [a + n for a, n in zip(starts, lengths)], g)
    k, v = c.read(table, _ends(lengths), rows, positions=_ints(starts) if any(starts) else None, dtype=dtype)
    for name, got in (("k", k), ("v", v)):
        want = torch.cat([gather(pool, name, table, b, torch.arange(a, a + n, device="cuda"), page) for b, (a, n) in enumerate(zip(starts, lengths))])
        assert torch.equal(got, want.float().to(dtype)), name     # exact in 64 bits, rounded once to fp32 and to the type


# ---------------------------------------------------------------------------------------------- decode

def _check_decode(c, pool, table, lengths, q, got, scale=None):
    for b, n in enumerate(lengths):
        if n == 0:
            assert not got[b].any()
            continue
        at = torch.arange(n, device="cuda")
        k, v = gather(pool, "k", table, b, at, c.page_size), gather(pool, "v", table, b, at, c.page_size)
        want, big, spread, mass = attend(q[b:b + 1], k, v, n - 1, scale)
        off, tol = (got[b:b + 1].double() - want).abs(), tolerance(q.dtype, want, big, spread, mass, c.head_dim)
        assert bool((off <= tol).all()), (b, n, float(off.max()), float((off / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,heads,share,page,lengths", [
    (128, 8, 4, 64, [1000]), (128, 1, 1, 16, [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129]), (64, 2, 7, 32, [0, 0, 5000, 33, 1, 700]),
    (64, 1, 16, 128, [300, 17]), (128, 2, 8, 16, [2049] * 3), (128, 4, 3, 64, [9, 4096, 0, 31] * 9), (64, 1, 1, 16, [40000]), (128, 1, 33, 64, [90, 0, 513])])
def test_decode_against_64_bits(cuda, dtype, hd, heads, share, page, lengths):
    g = _gen(8)
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in lengths) + 1, page, heads, heads * share, hd)
    pool = random_pool(c, g)
    table = random_table(c, lengths, g, width=max(1, -(-max(lengths) // page)) + 2)
    q = _randn(g, len(lengths), heads * share, hd, dtype=dtype) * 2
    _check_decode(c, pool, table, lengths, q, c.decode(q, table, _ints(lengths)))
    out = torch.empty_like(q)
    assert c.decode(q, table, _ints(lengths), scale=0.3, out=out) is out
    _check_decode(c, pool, table, lengths, q, out, 0.3)
    assert torch.equal(out, c.decode(q, table, _ints(lengths), scale=0.3))     # the same call gives the same bits
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,share,page,lengths", [(128, 8, 4, 64, [1000]), (64, 4, 7, 16, [5000, 333, 12000]), (128, 2, 16, 32, [2000] * 4)])
def test_fp32_decode_keeps_fp32_accuracy(cuda, hd, heads, share, page, lengths):
    """Over all results, errors add up as independent ones do.  Per score: operands of 22 bits (2^-23 each, two of them) and fp32 sums
    of hd products, 2^-24 sqrt(hd) of a product's size at random, which is 2^-24 sqrt(2) of the score's spread of about 1; weights
    of 22 bits and sums over tokens likewise.  Together below 2^-21 of a result; twice that is allowed."""
    g = _gen(20)
    c = ops.Q4PagedKVCache(sum(-(-n // page) for n in lengths), page, heads, heads * share, hd)
    pool = random_pool(c, g)
    table = random_table(c, lengths, g)
    q = _randn(g, len(lengths), heads * share, hd)
    got, off, size = c.decode(q, table, _ints(lengths)), 0.0, 0.0
    for b, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        want = attend(q[b:b + 1], *(gather(pool, x, table, b, at, page) for x in ("k", "v")), n - 1)[0]
        off += float((got[b:b + 1].double() - want).square().sum())
        size += float(want.square().sum())
    assert (off / size) ** 0.5 <= 2.0 ** -20, (off / size) ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_sees_nothing_behind_the_lengths(cuda, dtype):
    """Pages end inside a tile, and what is behind the last token is NaN."""
    g, lengths = _gen(9), [5, 16, 30, 75]
    c = ops.Q4PagedKVCache(20, 16, 2, 8, 128)
    pool = random_pool(c, g)
    table = random_table(c, lengths, g)
    q = _randn(g, 4, 8, 128, dtype=dtype)
    want = c.decode(q, table, _ints(lengths))
    for n in POOL:
        if n.endswith("codes"):
            continue
        keep = torch.zeros(pool[n].shape[:3], dtype=torch.bool, device=cuda)
        for b, m in enumerate(lengths):
            at = torch.arange(m, device=cuda)
            keep[table[b].long()[at // 16], :, at % 16] = True
        pool[n][~keep] = float("nan")
    c.load(**pool)
    assert torch.equal(c.decode(q, table, _ints(lengths)), want)


@pytest.mark.gpu
def test_decode_extremes(cuda):
    """Scores that differ by hundreds, a query of zeros, NaN in a query and in a key that is seen."""
    g = _gen(10)
    c = ops.Q4PagedKVCache(8, 64, 1, 4, 128)
    pool = random_pool(c, g)
    table = random_table(c, [500], g)
    q = _randn(g, 1, 4, 128)
    q[0, 0] *= 100
    q[0, 1] = 0
    _check_decode(c, pool, table, [500], q, c.decode(q, table, _ints([500])))
    q[0, 2, 7] = float("nan")
    got = c.decode(q, table, _ints([500]))
    assert torch.isnan(got[0, 2]).all() and torch.isfinite(got[0, [0, 1, 3]]).all()
    pool["k_mins"][table[0, 3].long(), 0, 9, 2] = float("nan")
    c.load(**pool)
    assert torch.isnan(c.decode(q, table, _ints([500]))).all()
    assert torch.isfinite(c.decode(q, table, _ints([201]))[0, [0, 1, 3]]).all()


@pytest.mark.gpu
def test_pages_beyond_four_gigabytes(cuda):
    c = ops.Q4PagedKVCache(56000, 64, 8, 8, 128, rope_theta=THETA)      # 81,920 bytes a page
    g, ids = _gen(11), [0, 55999, 27000, 52500]
    table = _ints([ids])
    k, v, q = _randn(g, 200, 8, 128), _randn(g, 200, 8, 128), _randn(g, 1, 8, 128)
    c.append(k, v, table, _ints([0]), cu_seqlens=_ends([200]))
    small = ops.Q4PagedKVCache(4, 64, 8, 8, 128, rope_theta=THETA)
    small.append(k, v, _ints([[0, 1, 2, 3]]), _ints([0]), cu_seqlens=_ends([200]))
    assert torch.equal(c.pool[ids], small.pool)
    assert torch.equal(c.decode(q, table, _ints([200])), small.decode(q, _ints([[0, 1, 2, 3]]), _ints([200])))
    for a, b in zip(c.read(table, _ends([200]), 200), small.read(_ints([[0, 1, 2, 3]]), _ends([200]), 200)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_captured_step_follows_tables_and_lengths(cuda):
    """append and decode in one graph, replayed with other tokens, tables and lengths; two graphs on two streams at a time."""
    g, page = _gen(12), 16
    lengths = [40, 7, 200]
    c = ops.Q4PagedKVCache(40, page, 2, 8, 64, rope_theta=THETA)
    random_pool(c, g)
    table = random_table(c, [300] * 2 + [16], g, width=20)
    graphs = []
    for _ in range(2):
        s = dict(k=_randn(g, 3, 2, 64), v=_randn(g, 3, 2, 64), q=_randn(g, 3, 8, 64), table=table.clone(), pos=_ints([0, 1, 2]), n=_ints([1, 2, 3]))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s["turned"] = c.append(s["k"], s["v"], s["table"], s["pos"], q=s["q"])
            s["out"] = c.decode(s["turned"], s["table"], s["n"])
        graphs.append((graph, s, side))
    table2 = random_table(c, lengths, g, width=20)
    for step in range(3):
        kept = c.pool.clone()
        pos = [n + step for n in lengths]
        new = dict(k=_randn(g, 3, 2, 64), v=_randn(g, 3, 2, 64), q=_randn(g, 3, 8, 64))
        turned = c.append(new["k"], new["v"], table2, _ints(pos), q=new["q"])
        want, pool = c.decode(turned, table2, _ints([p + 1 for p in pos])), c.pool.clone()
        c.pool.copy_(kept)
        torch.cuda.synchronize()
        for graph, s, side in graphs:       # both write the same, at the same time
            for n in ("k", "v", "q"):
                s[n].copy_(new[n])
            s["table"].copy_(table2)
            s["pos"].copy_(_ints(pos))
            s["n"].copy_(_ints([p + 1 for p in pos]))
        torch.cuda.synchronize()
        for graph, s, side in graphs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.pool, pool)
        for graph, s, side in graphs:
            assert torch.equal(s["out"], want) and torch.equal(s["turned"], turned)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(cuda):
    g, lengths = _gen(13), [3000, 100, 0, 777]
    c = ops.Q4PagedKVCache(80, 64, 4, 16, 128)
    random_pool(c, g)
    table, n = random_table(c, lengths, g), _ints(lengths)
    qs = [_randn(g, 4, 16, 128) for _ in range(2)]
    want = [c.decode(q, table, n) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(c.decode(qs[i], table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
