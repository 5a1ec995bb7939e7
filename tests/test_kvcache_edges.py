"""The E8-coded key/value cache without a GPU: what its entry points say to arguments that are none."""
import pytest
import torch


@pytest.mark.parametrize("q", [torch.zeros(()), torch.zeros(2, 2, 0), None, [1.0]], ids=["no dimension", "no values", "None", "a list"])
def test_queries_that_are_none_are_refused_like_others(q):
    """The default scale follows from the cache, not from q: a q that has no last dimension, or none at all, gets the refusal that names what is wrong."""
    from coset_b200 import kvcache as kv
    pages, s = torch.zeros(1, 2, 16, 18, dtype=torch.int32), torch.arange(2)
    with pytest.raises(ValueError, match="CUDA"):  # the pages are looked at first
        kv.e8_cache_attention(q, pages, s.int().view(2, 1), s.int())
