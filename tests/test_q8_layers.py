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
