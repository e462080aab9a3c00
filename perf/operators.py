"""Serving over a key/value cache held in 4 bits, as cases that can be timed: appending keys and values to the pages with the
position rotation on the way, attention of single tokens over the pages, attention over whole prompts of packed sequences, and
the two together for a prompt that arrives in chunks.

``listed()`` has the attention geometry of the benchmark configurations (32 query heads, 8 KV heads, head_dim 128) next to
other head layouts; ``draw(rng)`` spreads over the ranges around them.  With ``own`` the calls are the package's; without it
the same operators are spelled out in elementary torch operations.

The format of the cache: 32 consecutive dimensions of a token's key or value share a scale and a minimum in bf16,
``minimum = floor(min x)`` and ``scale = ceil((max x - minimum) / 15)``, floor and ceil to the neighbouring bf16 number, and
``x`` is held as ``round((x - minimum) / scale)`` in 4 bits."""
import math

import torch

own = False

GROUP = 32           # dimensions that share a scale and a minimum
THETA = 1e6          # base of the position rotation
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # A decoding step puts one token of one sequence into the cache: the smallest call.
        {"name": "append b1", "kind": "append", "batch": 1, "longest": 1, "past": 1000, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "f32"},
        # The same for a batch of sequences at positions of their own.
        {"name": "append b64", "kind": "append", "batch": 64, "longest": 1, "past": 5000, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "bf16"},
        # A long prompt, and packed prompts of very different lengths behind cached ones.
        {"name": "append prompt 16384", "kind": "append", "batch": 1, "longest": 16384, "past": 0, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "bf16"},
        {"name": "append ragged", "kind": "append", "batch": 24, "longest": 1111, "past": 301, "kv_heads": 4, "share": 7, "hd": 64, "page": 16, "dtype": "f32"},
        # Single tokens over the pages: a short chat, long contexts of a batch, contexts of all lengths (an empty one among them).
        {"name": "decode 1000 b1", "kind": "decode", "batch": 1, "longest": 1000, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "f32"},
        {"name": "decode 32768 b16", "kind": "decode", "batch": 16, "longest": 32768, "even": True, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "bf16"},
        {"name": "decode ragged b48", "kind": "decode", "batch": 48, "longest": 20011, "kv_heads": 4, "share": 7, "hd": 64, "page": 16, "dtype": "f32"},
        # Whole prompts: a few words, a document, packed prompts of all lengths, and fp32 activations.
        {"name": "prompt 37", "kind": "prompt", "batch": 1, "longest": 37, "kv_heads": 8, "share": 4, "hd": 128, "dtype": "bf16"},
        {"name": "prompt 8192", "kind": "prompt", "batch": 1, "longest": 8192, "kv_heads": 8, "share": 4, "hd": 128, "dtype": "bf16"},
        {"name": "prompt ragged", "kind": "prompt", "batch": 20, "longest": 2003, "kv_heads": 4, "share": 7, "hd": 64, "dtype": "bf16"},
        {"name": "prompt f32 2048", "kind": "prompt", "batch": 2, "longest": 2048, "even": True, "kv_heads": 8, "share": 4, "hd": 128, "dtype": "f32"},
        # A prompt that comes in chunks: 1024 positions behind 7000 cached ones, through the cache and its attention.
        {"name": "chunk 1024 after 7000", "kind": "chunk", "batch": 2, "longest": 1024, "even": True, "past": 7000, "kv_heads": 8, "share": 4, "hd": 128, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "prompt", "prompt", "chunk"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16"]), "kv_heads": rng.choice([1, 2, 4, 8, 8]),
         "share": rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), "hd": rng.choice([64, 128, 128]), "even": rng.random() < 0.4}
    heads = c["kv_heads"] * c["share"]
    if kind != "prompt":
        c["page"] = rng.choice([16, 32, 64, 64, 128])
    if kind == "append":
        c["past"] = _log(rng, 1, 16000)
        c["batch"] = _log(rng, 1, 128)
        c["longest"] = 1 if rng.random() < 0.4 else _log(rng, 2, min(16384, 16384 * 32 // (c["batch"] * heads)))
    elif kind == "decode":
        c["batch"] = _log(rng, 1, 128)
        c["longest"] = _log(rng, 1, min(131072, 16 * 32768 * 8 // (c["batch"] * c["kv_heads"] * max(1, c["share"] // 4))))
    elif kind == "prompt":
        c["batch"] = _log(rng, 1, 32)
        c["longest"] = _log(rng, 1, int((8192 * 8192 * 32 / (4 if c["dtype"] == "f32" else 1) / (c["batch"] * heads)) ** 0.5))
    else:
        c["batch"] = _log(rng, 1, 8)
        c["longest"] = _log(rng, 2, 1024)
        c["past"] = _log(rng, 1, 12000)
        most = 2 * 7000 * 1024 * 32 // (4 if c["dtype"] == "f32" else 1) // (c["batch"] * heads)
        c["longest"] = max(2, min(c["longest"], int(most ** 0.5)))
        c["past"] = max(1, min(c["past"], most // c["longest"] - c["longest"]))
    return c


# ---------------------------------------------------------------------------------------------- inputs

def _lengths(c):
    """Tokens of every sequence: all the longest, or from one up to it with an empty sequence among eight or more."""
    n, longest = c["batch"], c["longest"]
    if c.get("even") or longest == 1 or n == 1:
        return [longest] * n
    spread = [max(1, longest * (i + 1) ** 2 // n ** 2) for i in range(n)]
    if n >= 8:
        spread[1] = 0
    return [spread[i * 5 % n] if n % 5 else spread[i] for i in range(n)]


def _pasts(c):
    """Tokens that every sequence has in the cache before the call."""
    return [max(0, c["past"] - 3 * i) if c["kind"] == "chunk" else (c["past"] * (i + 1)) // c["batch"] for i in range(c["batch"])]


def _ends(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, c, totals):
    """The pages of a cache with room for ``totals`` tokens: codes as whole numbers, scales and minima as a layer's keys and
    values of unit variance have them, and a block table that scatters the sequences over the pages."""
    page, heads, hd = c["page"], c["kv_heads"], c["hd"]
    counts = [-(-n // page) for n in totals]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(totals), max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    ends = _ends(counts)
    for b, n in enumerate(counts):
        table[b, :n] = order[ends[b]:ends[b] + n]
    pools = {}
    for name in ("k", "v"):
        shape = (pages, heads, page, hd // GROUP)
        pools[name + "_codes"] = torch.randint(0, 16, (pages, heads, page, hd), generator=g, device="cuda", dtype=torch.uint8)
        pools[name + "_scales"] = (0.27 + 0.04 * torch.randn(shape, generator=g, device="cuda")).abs().to(torch.bfloat16)
        pools[name + "_mins"] = (-2.0 + 0.4 * torch.randn(shape, generator=g, device="cuda")).to(torch.bfloat16)
    return table, pools


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 29)
    dtype, kind, hd = DTYPES[c["dtype"]], c["kind"], c["hd"]
    lengths = _lengths(c)
    randn = lambda tokens, heads, scale: (torch.randn(tokens, heads, hd, generator=g, device="cuda") * scale).to(dtype)  # noqa: E731
    s = {"case": c, "longest": max(lengths)}
    q_heads, rows = c["kv_heads"] * c["share"], c["batch"] if kind == "decode" else sum(lengths)
    s["q"] = randn(rows, q_heads, 1.0)
    if kind != "decode":
        s["k"], s["v"] = randn(rows, c["kv_heads"], 1.0), randn(rows, c["kv_heads"], 1.0)
        s["ends"] = _ints(_ends(lengths))
    if kind == "decode":
        totals = lengths
        s["lengths"] = _ints(lengths)
    elif kind != "prompt":
        pasts = _pasts(c)
        totals = [p + n for p, n in zip(pasts, lengths)]
        s["positions"] = _ints(pasts)
        s["total_ends"], s["total"] = _ints(_ends(totals)), sum(totals)
    if kind != "prompt":
        s["most"] = max(totals)
        s["table"], pools = _cache(g, c, totals)
        if own:
            from ojasx_b200 import ops
            s["cache"] = ops.Q4PagedKVCache(pools["k_codes"].shape[0], c["page"], c["kv_heads"], q_heads, hd, rope_theta=THETA)
            s["cache"].load(**pools)
        else:
            s["pools"] = pools
    return s


# ---------------------------------------------------------------------------------------------- the framework's operators

def _run_own(s):
    from ojasx_b200 import ops
    c, kind = s["case"], s["case"]["kind"]
    if kind == "append":
        single = c["longest"] == 1
        q = s["cache"].append(s["k"], s["v"], s["table"], s["positions"], q=s["q"], cu_seqlens=None if single else s["ends"])
        return (q,) + s["cache"].read(s["table"], s["ends"], s["k"].shape[0], positions=s["positions"])
    if kind == "decode":
        return s["cache"].decode(s["q"], s["table"], s["lengths"])
    if kind == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], s["ends"])
    out = s["cache"].prefill(s["q"], s["k"], s["v"], s["table"], s["positions"], s["ends"], s["total_ends"], s["total"])
    return (out,) + s["cache"].read(s["table"], s["ends"], s["k"].shape[0], positions=s["positions"])


# ---------------------------------------------------------------------------------------------- the same in plain form

def _owners(ends, rows):
    """Sequence of every packed row, and the row's place in it."""
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(ends[1:].long(), at, right=True)
    return seq, at - ends.long()[seq]


def _rotate(x, positions):
    """Dimensions j and j + hd/2 turned by position * theta^(-2j/hd), the angles in 64 bits."""
    half = x.shape[-1] // 2
    rates = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = positions.double()[:, None, None] * rates
    cos, sin = torch.cos(angle), torch.sin(angle)
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).float()


def _floor_bf16(x):
    """The largest bf16 number that is not above x."""
    bits = x.view(torch.int32)
    cut = bits & -65536
    return torch.where((bits < 0) & (cut != bits), cut + 65536, cut).view(torch.float32)


def _quantize(x):
    """(codes, scales, minima) of fp32 vectors [..., hd]."""
    x = x.unflatten(-1, (-1, GROUP))
    low = _floor_bf16(x.amin(-1))
    scale = -_floor_bf16(-((x.amax(-1) - low) / torch.full_like(low, 15)))    # (by a number, torch multiplies by its reciprocal)
    codes = torch.round((x - low[..., None]) / scale[..., None].clamp(min=1e-30)).clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), scale.to(torch.bfloat16), low.to(torch.bfloat16)


def _value(pools, name, page, at):
    """fp32 values of cached tokens: page ids and places in the page, of any shape."""
    codes = pools[name + "_codes"][page, :, at].float().unflatten(-1, (-1, GROUP))
    return (codes * pools[name + "_scales"][page, :, at].float()[..., None] + pools[name + "_mins"][page, :, at].float()[..., None]).flatten(-2)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(hd)) v in fp32; q [B, Hkv, share, Lq, hd], k and v [B, Hkv, Lk, hd], seen [B, Lq, Lk].  A row that
    sees nothing is zero."""
    B, H, share, Lq, hd = q.shape
    score = (q.reshape(B, H, share * Lq, hd) @ k.transpose(-1, -2)).view(B, H, share, Lq, -1)
    score.mul_(hd ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(B, H, share * Lq, -1) @ v).view(B, H, share, Lq, hd)
    return out / total.clamp(min=1e-30)


def _packed(s, q, k, v, ends, key_ends, dtype):
    """Causal attention of packed sequences, padded to the longest; the last queries see the last keys."""
    c = s["case"]
    most = s["longest"] if key_ends is ends else s["most"]
    n, nk = ends[1:] - ends[:-1], key_ends[1:] - key_ends[:-1]
    row, col = torch.arange(s["longest"], device="cuda"), torch.arange(most, device="cuda")
    place = lambda e, at, rows: (e[:-1, None] + at).clamp(max=rows - 1).long()  # noqa: E731
    qp = q[place(ends, row, q.shape[0])].float().unflatten(2, (c["kv_heads"], c["share"])).permute(0, 2, 3, 1, 4)
    kp, vp = (t[place(key_ends, col, t.shape[0])].float().transpose(1, 2) for t in (k, v))
    seen = (col < nk[:, None])[:, None, :] & (col <= row[:, None] + (nk - n)[:, None, None])
    out = _attend(qp, kp, vp, seen).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[_owners(ends, q.shape[0])].to(dtype)


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    dtype = DTYPES[c["dtype"]]
    if kind == "prompt":
        return _packed(s, s["q"], s["k"], s["v"], s["ends"], s["ends"], dtype)
    page, pools, table = c["page"], s["pools"], s["table"].clamp(min=0).long()
    if kind == "decode":
        at = torch.arange(s["most"], device="cuda")
        k, v = (_value(pools, name, table[:, at // page], at % page).transpose(1, 2) for name in ("k", "v"))
        q = s["q"].float().unflatten(1, (c["kv_heads"], c["share"]))[:, :, :, None]
        return _attend(q, k, v, (at < s["lengths"][:, None])[:, None]).squeeze(3).flatten(1, 2).to(dtype)
    rows = s["k"].shape[0]
    seq, place = _owners(s["ends"], rows)
    pos = s["positions"].long()[seq] + place
    ids, at = table[seq, pos // page], pos % page
    q = _rotate(s["q"].float(), pos).to(dtype)
    for name, x in (("k", _rotate(s["k"].float(), pos)), ("v", s["v"].float())):
        for part, value in zip(("_codes", "_scales", "_mins"), _quantize(x)):
            pools[name + part][ids, :, at] = value
    new = tuple(_value(pools, name, ids, at).to(torch.bfloat16) for name in ("k", "v"))
    if kind == "append":
        return (q,) + new
    # the operators in turn, each rounding what it gives to the activations' type: the turned queries, the values that are
    # read back, and the attention over them
    seq, place = _owners(s["total_ends"], s["total"])
    ids, at = table[seq, place // page], place % page
    k, v = (_value(pools, name, ids, at).to(dtype) for name in ("k", "v"))
    return (_packed(s, q, k, v, s["ends"], s["total_ends"], dtype),) + new


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---------------------------------------------------------------------------------------------- work and the exact results

def work(case):
    """A cached value has 5 bits (its code and its share of a scale and a minimum)."""
    c, size = case, 4 if case["dtype"] == "f32" else 2
    lengths, hd, kv, heads = _lengths(c), c["hd"], c["kv_heads"], c["kv_heads"] * c["share"]
    rows, kind = sum(lengths), c["kind"]
    if kind == "decode":
        return {"bytes": 2 * kv * hd * 5 / 8 * rows + 2 * size * c["batch"] * heads * hd, "flops": 4 * heads * hd * rows}
    pasts = _pasts(c) if "past" in c else [0] * len(lengths)
    pairs = sum(p * n + n * (n + 1) // 2 for p, n in zip(pasts, lengths))
    if kind == "prompt":
        return {"bytes": 2 * size * rows * (heads + kv) * hd, "flops": 4 * heads * hd * pairs}
    # new keys and values in, their codes out, and read back as bf16
    bytes_ = rows * hd * (2 * kv * (size + 5 / 8) + 2 * size * heads + 2 * kv * (5 / 8 + 2))
    if kind == "append":
        return {"bytes": bytes_, "flops": rows * hd * (3 * heads + 9 * kv)}
    return {"bytes": bytes_ + sum(pasts) * 2 * kv * hd * 5 / 8, "flops": 4 * heads * hd * pairs}


def _exact_quantized(x):
    """What the cache's format makes of 64-bit vectors [..., hd]: minimum and scale are whole multiples of a power of two,
    2^-7 of the largest one below their size."""
    def step(y):
        return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1e-300))) - 7)
    groups = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    low = groups.min(-1).values
    low = torch.floor(low / step(low)) * step(low)
    scale = (groups.max(-1).values - low) / torch.full_like(low, 15)
    scale = torch.ceil(scale / step(scale)) * step(scale)
    codes = ((groups - low[..., None]) / scale[..., None].clamp(min=1e-300)).round().clamp(0, 15)
    return (low[..., None] + codes * scale[..., None]).reshape(x.shape)


def _exact_values(state_pools, name, ids, at):
    codes, scales, mins = (state_pools[name + part][ids, :, at].double() for part in ("_codes", "_scales", "_mins"))
    return codes * scales.repeat_interleave(GROUP, -1) + mins.repeat_interleave(GROUP, -1)


def _exact_attention(q, k, v, first):
    """One sequence: q [n, H, hd], k and v [m, Hkv, hd]; query i sees the keys up to first + i.  Query rows in slices."""
    n, H, hd = q.shape
    share, out = H // k.shape[1], torch.empty_like(q)
    rows = max(1, 2 ** 27 // max(1, share * k.shape[0]))
    for h in range(H // share):
        for i in range(0, n, rows):
            part = q[i:i + rows, h * share:(h + 1) * share]
            logits = torch.einsum("ird,md->irm", part, k[:, h]) / math.sqrt(hd)
            hidden = torch.arange(k.shape[0], device="cuda") > first + torch.arange(i, i + part.shape[0], device="cuda")[:, None]
            weights = torch.softmax(logits.masked_fill(hidden[:, None], -math.inf), -1)
            out[i:i + rows, h * share:(h + 1) * share] = torch.einsum("irm,md->ird", weights, v[:, h])
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    c, kind, hd = case, case["kind"], case["hd"]
    lengths = _lengths(c)
    ends = _ends(lengths)
    if kind == "prompt":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        parts = [_exact_attention(q[a:b], k[a:b], v[a:b], 0) for a, b in zip(ends, ends[1:]) if b > a]
        return torch.cat(parts)
    spot = lambda b, t: (s["table"][b].long()[t // c["page"]], t % c["page"])  # noqa: E731
    if kind == "decode":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            if n:
                ids, at = spot(b, torch.arange(n, device="cuda"))
                k, v = _exact_values(s["pools"], "k", ids, at), _exact_values(s["pools"], "v", ids, at)
                out[b:b + 1] = _exact_attention(s["q"][b:b + 1].double(), k, v, n - 1)
        return out
    pasts = _pasts(c)

    def turned(x):
        at = torch.cat([torch.arange(p, p + n, dtype=torch.float64, device="cuda") for p, n in zip(pasts, lengths)])
        # a pair of dimensions as one complex number, turned by a power of theta^(2 / hd)
        pairs = torch.complex(x[..., :hd // 2].double(), x[..., hd // 2:].double())
        power = torch.exp(torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") * (-math.log(THETA) / hd))
        pairs = pairs * torch.polar(torch.ones_like(at[:, None] * power), at[:, None] * power)[:, None]
        return torch.cat((pairs.real, pairs.imag), -1)

    q, k, v = turned(s["q"]), _exact_quantized(turned(s["k"])), _exact_quantized(s["v"].double())
    if kind == "append":
        return q, k, v
    out = torch.empty_like(q)
    for b, (a, e) in enumerate(zip(ends, ends[1:])):
        ids, at = spot(b, torch.arange(pasts[b], device="cuda"))
        ks = torch.cat((_exact_values(s["pools"], "k", ids, at), k[a:e]))
        vs = torch.cat((_exact_values(s["pools"], "v", ids, at), v[a:e]))
        if e > a:
            out[a:e] = _exact_attention(q[a:e], ks, vs, pasts[b])
    return out, k, v
