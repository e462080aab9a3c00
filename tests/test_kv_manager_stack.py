"""The cache manager over decoder stacks and bare 4-bit caches: what it reports is what the next step sees."""
import pytest
import torch

from ojasx_b200 import inference_engine as ie
from ojasx_b200 import ops
from ojasx_b200.kv_cache import OjasXKVCacheManager

CFG = dict(layers=2, hidden=256, q_heads=4, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=64, vocab=512, max_seq_len=100, distinct_layers=2, page_size=16)


def _bare():
    """A 4-bit cache without its pages: the manager looks at its type and size alone."""
    c = ops.Q4PagedKVCache.__new__(ops.Q4PagedKVCache)
    c.pool = torch.zeros(2, 80, dtype=torch.uint8)
    return c


def test_bare_4_bit_caches_need_their_lengths():
    for held in (_bare(), [_bare(), _bare()], {"layer": (_bare(),)}):
        m = OjasXKVCacheManager(max_context_length=50)
        with pytest.raises(ValueError, match="sequence_length"):
            m.update(held)
        assert m.past_key_values is None
        m.update(held, sequence_length=40)
        assert m.sequence_length == 40
        with pytest.raises(ValueError, match="caller's"):
            m.crop(39)
        assert m.sequence_length == 40
        m.crop(40)
        m.update(held, sequence_length=39)
        assert m.sequence_length == 39
        with pytest.raises(ValueError, match="admission bound"):
            m.update(held, sequence_length=51)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_format", ["q4", "vq"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_a_cropped_stack_goes_on_from_there(cuda, kv_format, use_graph):
    """A stack that went further and was cropped gives the bits of one that did not."""
    cfg = ie.StackConfig(**CFG, kv_format=kv_format)
    weights = ie.make_stack_weights(3, cfg)
    a, b = (ie.VQDecoderStack(weights, cfg, 2, torch.float32, use_graph=use_graph) for _ in range(2))
    ids = torch.randint(0, CFG["vocab"], (2, 40), generator=torch.Generator().manual_seed(5))
    a.prefill(ids[:, :32], batched=False)
    m = OjasXKVCacheManager(max_context_length=64)
    m.update(a)
    assert m.sequence_length == 32
    with pytest.raises(ValueError, match="admission bound"):
        OjasXKVCacheManager(max_context_length=31).update(a)
    m.crop(64)
    assert m.sequence_length == a.position == 32
    m.crop(10)
    assert m.sequence_length == a.position == 10 and a.pos.tolist() == [10, 10] and a.lengths.tolist() == [11, 11]
    b.prefill(ids[:, :10], batched=False)
    for t in range(10, 14):
        other = (ids[:, t] + 1) % CFG["vocab"]
        assert torch.equal(a.decode_step(other), b.decode_step(other)), t
    assert m.sequence_length == a.position == 14
    assert torch.equal(a.prefill(ids[:, 14:30]), b.prefill(ids[:, 14:30]))
    with pytest.raises(ValueError):
        a.crop(-1)
    assert a.crop(0) == 0 and b.crop(3) == 3
    b.crop(0)
    assert torch.equal(a.generate(ids[:, :5], 3), b.generate(ids[:, :5], 3))
    m.reset()
    assert m.past_key_values is None and a.position == 0
