"""The decoder stack over 4-bit paged caches: prompts whole and token by token, captured steps, what the attention gives, and the
manager's accounting."""
import pytest
import torch

from ojasx_b200 import inference_engine as ie
from ojasx_b200 import ops
from ojasx_b200.kv_cache import OjasXKVCacheManager

from q4_plain import attend, gather, tolerance

CFG = dict(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=64, vocab=512, max_seq_len=100, distinct_layers=2,
           kv_format="q4", page_size=16)


def _stack(dtype=torch.float32, batch=2, use_graph=False, **kw):
    cfg = ie.StackConfig(**{**CFG, **kw})
    return ie.VQDecoderStack(ie.make_stack_weights(3, cfg), cfg, batch, dtype, use_graph=use_graph)


def _ids(batch, n, seed=0):
    return torch.randint(0, CFG["vocab"], (batch, n), generator=torch.Generator().manual_seed(seed))


def test_formats_are_checked():
    with pytest.raises(ValueError):
        ie.VQDecoderStack(None, ie.StackConfig(kv_format="q8"))
    with pytest.raises(ValueError):
        ie.VQDecoderStack(None, ie.StackConfig(kv_format="q4"), segment=object())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_whole_in_chunks_and_token_by_token(cuda, dtype):
    """The same prompt three ways: linears and experts keep their bits in fp32, attention its tolerance of about 2^-16, and a code that
    lies that near to a border may be the next one, a step of one value of one token: 2 % of the largest logit are far above either.
    bf16 kernels for batches add in other orders, layer by layer: 2^-8 a rounding, eight roundings a layer."""
    ids = _ids(2, 37)
    bound = 0.02 if dtype == torch.float32 else 0.15
    a, b, c = _stack(dtype), _stack(dtype), _stack(dtype)
    la, lb, lc = a.prefill(ids), b.prefill(ids, batched=False), c.prefill(ids, max_rows=20)
    top = float(la.abs().max())
    assert la.shape == lb.shape == lc.shape == (2, CFG["vocab"])
    assert float((la - lb).abs().max()) <= bound * top and float((la - lc).abs().max()) <= bound * top
    assert a.position == b.position == c.position == 37
    for s in (a, b, c):
        assert s.pos.tolist() == [37, 37] and s.lengths.tolist() == [38, 38]
    na, nb = a.decode_step(la.argmax(-1)), b.decode_step(la.argmax(-1))
    assert float((na - nb).abs().max()) <= bound * float(na.abs().max())
    for l in a.layers:
        l.cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 3])
def test_captured_steps_give_the_bits_of_eager_ones(cuda, batch):
    a, b = _stack(batch=batch), _stack(batch=batch, use_graph=True)
    ids = _ids(batch, 20, seed=1)
    assert torch.equal(a.prefill(ids[:, :9]), b.prefill(ids[:, :9]))
    for t in range(9, 20):
        assert torch.equal(a.decode_step(ids[:, t]), b.decode_step(ids[:, t])), t
    for x, y in zip(a.layers, b.layers):
        assert torch.equal(x.cache.pool, y.cache.pool)
    a.reset()
    b.reset()
    assert torch.equal(a.generate(ids[:, :5], 4), b.generate(ids[:, :5], 4))


@pytest.mark.gpu
def test_attention_of_a_step_is_that_over_the_pages(cuda):
    s = _stack()
    s.prefill(_ids(2, 30, seed=2))
    seen = []
    decode = ops.Q4PagedKVCache.decode

    def watch(self, q, table, lengths, *a, **kw):
        out = decode(self, q, table, lengths, *a, **kw)
        seen.append((self, q.clone(), lengths.clone(), out.clone()))
        return out

    ops.Q4PagedKVCache.decode = watch
    try:
        s.decode_step(torch.tensor([5, 6]))
    finally:
        ops.Q4PagedKVCache.decode = decode
    assert len(seen) == 2
    for cache, q, lengths, out in seen:
        assert lengths.tolist() == [31, 31]
        pool = cache.unload()
        for b in range(2):
            k, v = (gather(pool, n, s.block_table, b, torch.arange(31, device="cuda"), 16) for n in ("k", "v"))
            want, big, spread, mass = attend(q[b:b + 1], k, v, 30)
            assert bool(((out[b:b + 1].double() - want).abs() <= tolerance(q.dtype, want, big, spread, mass, 64)).all())


@pytest.mark.gpu
def test_full_caches_are_refused_and_the_manager_counts_pages(cuda):
    s = _stack(max_seq_len=32)
    s.prefill(_ids(2, 31))
    s.decode_step(torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        s.decode_step(torch.tensor([1, 2]))
    m = OjasXKVCacheManager(max_context_length=64)
    m.update(s, sequence_length=32)
    stats = m.stats()
    assert stats.dtype == "uint4_groups" and stats.num_cached_layers == 2 and stats.sequence_length == 32
    assert stats.allocated_bytes == 2 * 2 * 2 * 2 * 16 * 80     # layers, sequences, pages, KV heads, tokens, bytes at head_dim 64
    m.crop(10)
    assert m.sequence_length == 10
    with pytest.raises(ValueError):
        m.update(s, sequence_length=65)
