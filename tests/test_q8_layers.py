"""Which layers, pages and callers may have the cache in 8 bits: no GPU needed."""
import pytest
import torch

from kllm_b200 import kernels


def test_pages_that_the_append_does_not_take():
    from kllm_b200.cache.manager import CacheManager
    from kllm_b200.parts.spec import PagedKVNeed, StateNeed
    need, f8 = PagedKVNeed(2, 64, eight_bits=True), torch.float8_e4m3fn
    most = kernels.Q8_MAX_PAGE
    CacheManager([need], most, 2, max_requests=1, dtype=torch.bfloat16, cache_dtype=f8)
    with pytest.raises(ValueError, match=f"pages of {most + 1} tokens"):
        CacheManager([need], most + 1, 2, max_requests=1, dtype=torch.bfloat16, cache_dtype=f8)
    with pytest.raises(ValueError, match="pages of 8192 tokens"):
        CacheManager.pages_within([need], 8192, torch.bfloat16, 2 ** 30, f8)
    # where there is nothing of the kind, the size is the user's
    CacheManager([need], most + 1, 2, max_requests=1, dtype=torch.bfloat16)
    CacheManager([StateNeed((8,), "float32")], most + 1, 2, max_requests=1, dtype=torch.bfloat16, cache_dtype=f8)


CFG = {"architectures": ["LlamaForCausalLM"], "num_hidden_layers": 3, "hidden_size": 64, "num_attention_heads": 4, "num_key_value_heads": 2,
       "head_dim": 32, "intermediate_size": 64, "vocab_size": 64, "max_position_embeddings": 64}


def shared_slot(reader=None, wrap=None):
    """A model whose first layer writes a cache that its second one reads; ``wrap`` stands for the blocks of other arrangements."""
    from kllm_b200 import models  # noqa: F401
    from kllm_b200.config.base import build_model_spec, parse_config
    from kllm_b200.parts.model import DecoderModel
    from kllm_b200.parts.spec import LayerCall
    spec = build_model_spec(parse_config(CFG))
    spec.blocks[1].mixer.params.update(reader or {})
    spec.schedule = [LayerCall(0, 0), LayerCall(1, 0, writes_cache=False), LayerCall(2, 1)]
    model = DecoderModel(spec, torch.float32, "cpu")
    if wrap is not None:
        model.blocks = [wrap(i, b) for i, b in enumerate(model.blocks)]
    return model


def taken(need):
    from kllm_b200.parts.spec import PagedKVNeed
    return [n.eight_bits for n in (need if isinstance(need, list) else [need]) if isinstance(n, PagedKVNeed)]


class Beside:
    """A block that keeps a state beside its mixer's cache, as some arrangements do."""

    def __init__(self, block):
        self.block = block

    def cache_need(self):
        from kllm_b200.parts.spec import StateNeed
        return [self.block.mixer.cache_need(), StateNeed((4,), "float32")]


class Bare:
    """A block without a mixer of its own that reads what another one wrote."""


@pytest.mark.parametrize("writer", [lambda b: b, Beside])
@pytest.mark.parametrize("reader", [lambda b: b, Beside])
def test_every_reader_of_a_slot_is_asked(writer, reader):
    wrap = lambda i, b: writer(b) if i == 0 else reader(b) if i == 1 else b  # noqa: E731
    assert [taken(n) for n in shared_slot(None, wrap).cache_needs()] == [[True], [True]]
    assert [taken(n) for n in shared_slot(dict(score_slopes="geometric"), wrap).cache_needs()] == [[False], [True]]


def test_a_reader_without_a_mixer_does_not_take_it():
    model = shared_slot(None, lambda i, b: Bare() if i == 1 else b)
    assert [taken(n) for n in model.cache_needs()] == [[False], [True]]


def test_a_layers_view_is_built_as_before():
    """Positions of the fields that were there before the scales."""
    from kllm_b200.parts.context import LayerCache
    states = {"conv": torch.zeros(1)}
    c = LayerCache(None, None, None, None, True, 16, states)
    assert c.page_size == 16 and c.states is states and c.k_scale is None and c.v_scale is None
