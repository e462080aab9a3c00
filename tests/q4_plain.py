"""Plain 64-bit forms of the 4-bit cache's format and of causal attention over packed sequences, for the tests of their kernels."""
import math

import torch

GROUP = 32


def floor_bf16(x):
    """The largest bf16 number not above an fp32 one."""
    y = x.to(torch.bfloat16)
    bits = y.view(torch.int16)
    lower = torch.where(bits >= 0, torch.where(bits == 0, torch.full_like(bits, -32767), bits - 1), bits + 1).view(torch.bfloat16)
    return torch.where(y.float() > x, lower, y)


def quantize(x):
    """(codes, scales, minima) of fp32 vectors [..., hd]; every operation is one that IEEE arithmetic rounds."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low = floor_bf16(g.amin(-1)).float()
    scale = (-floor_bf16(-((g.amax(-1) - low) / torch.full_like(low, 15)))).float()
    codes = torch.round((g - low[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), scale.to(torch.bfloat16), low.to(torch.bfloat16)


def values(codes, scales, mins):
    """What codes stand for, in 64 bits."""
    g = codes.double().unflatten(-1, (-1, GROUP))
    return (g * scales.double()[..., None] + mins.double()[..., None]).flatten(-2)


def rotate(x, positions, theta):
    """Dimensions j and j + hd/2 of [tokens, heads, hd] turned by position * theta^(-2j/hd), in 64 bits."""
    half = x.shape[-1] // 2
    angle = positions.double()[:, None, None] * theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)


def random_pool(cache, g):
    """Random codes, scales and minima for every token of a cache, loaded into it."""
    shape = (cache.num_pages, cache.kv_heads, cache.page_size)
    pool = {}
    for n in ("k", "v"):
        pool[n + "_codes"] = torch.randint(0, 16, (*shape, cache.head_dim), generator=g, device="cuda", dtype=torch.uint8)
        pool[n + "_scales"] = (torch.rand(*shape, cache.head_dim // GROUP, generator=g, device="cuda") * 0.3 + 0.02).to(torch.bfloat16)
        pool[n + "_mins"] = (torch.randn(*shape, cache.head_dim // GROUP, generator=g, device="cuda") - 1.5).to(torch.bfloat16)
    cache.load(**pool)
    return pool


def random_table(cache, lengths, g, width=None):
    """A block table that scatters sequences of the given lengths over the pool's pages; -1 where a sequence has none."""
    counts = [-(-n // cache.page_size) for n in lengths]
    order = torch.randperm(cache.num_pages, generator=g, device="cuda").to(torch.int32)
    assert sum(counts) <= cache.num_pages
    table = torch.full((len(lengths), width or max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def gather(pool, name, table, b, tokens, page):
    """64-bit values [n, kv_heads, hd] of a sequence's cached tokens."""
    ids = table[b].long()[tokens // page]
    return values(*(pool[name + part][ids, :, tokens % page] for part in ("_codes", "_scales", "_mins")))


def attend(q, k, v, first, scale=None):
    """One sequence in 64 bits: q [n, H, hd], k and v [m, Hkv, hd], query i sees the keys up to first + i.  Returns the result, the
    largest size of a value seen, sum p |v|, and the largest sum |q||k| * scale over the keys a query sees."""
    n, H, hd = q.shape
    share, m = H // k.shape[1], k.shape[0]
    if m == 0:
        zero = q.double() * 0
        return zero, 0.0, zero, zero[..., :1]
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    seen = torch.arange(m, device=q.device) <= first + torch.arange(n, device=q.device)[:, None]
    # what a query does not see has no part in its row, not even as 0 * inf: those places hold zeros, per row
    kk, vv = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = torch.einsum("nhd,mhd->hnm", q, kk) * scale
    s = torch.where(seen, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    if m and not bool(torch.isfinite(vv).all()):
        out = torch.stack([torch.where(seen[i][:, None, None], p[:, i].t()[:, :, None] * vv, 0.0).sum(0) for i in range(n)]) if n else q
    else:
        out = torch.einsum("hnm,mhd->nhd", p, vv)
    spread = torch.einsum("hnm,mhd->nhd", p, vv.abs().nan_to_num(0, 0, 0))
    big = torch.where(seen[:, :, None, None], vv.abs()[None].nan_to_num(0, 0, 0), 0.0).amax(1).amax(-1, keepdim=True) if n * m * H * hd < 2e8 else vv.abs().max()
    mass = torch.where(seen, torch.einsum("nhd,mhd->hnm", q.abs(), kk.abs()) * scale, 0.0).amax(-1).t()[:, :, None]
    return out, big, spread, mass


def tolerance(dtype, want, big, spread, mass, hd):
    """How far a kernel may be from the 64-bit result.  A score is a sum of hd products in fp32, summed in any order by adders that
    may cut a bit more than they should: its error is at most (hd + 8) * 2^-23 of the sum of sizes (`mass`, with the scale).  An
    error d of the scores changes weights by a factor of up to e^2d, the result by up to 2 d * big; the fp32 exponential of a score
    of size up to `mass` adds 2^-22 of it relative to the weight (its argument is rounded), and the sums over the weights 2^-20.
    bf16 results also have weights rounded to bf16 (half a step, 2^-8, of sum p |v|) and their own rounding (2^-8 of the value)."""
    d = mass * ((hd + 8) * 2.0 ** -23 + 2.0 ** -22)
    t = big * (2 * d + 2.0 ** -20) + 1e-30
    if dtype == torch.bfloat16:
        t = t + 2.0 ** -8 * spread + 2.0 ** -8 * want.abs()
    return t
