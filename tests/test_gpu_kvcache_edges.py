"""The E8-coded key/value cache at the edges of what its calls allow: layouts with dimensions of one."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_kvcache import DTYPES, api, as_words, expected_pages, rows

pytestmark = pytest.mark.gpu


def cut_from_wider(x, odd):
    """x [n, heads, dim] as a part of a projection whose rows are `odd` values wider, and so begin at no multiple of 16 bytes."""
    n, heads, dim = x.shape
    wide = torch.zeros(n, heads, dim + odd, dtype=x.dtype, device="cuda")
    wide[..., :dim] = x.cuda()
    return wide[..., :dim]


# ------------------------------------------------------------------ layouts
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim, heads, n", [(128, 1, 1), (64, 3, 1), (256, 1, 5), (128, 2, 4)])
def test_rows_of_any_stride_where_a_dimension_is_one(dim, heads, n, dtype):
    """A single token, or a single head, cut from rows of an odd length: the stride of a dimension of one is no multiple of 16 bytes, and means nothing."""
    kv = api()
    k, v = rows(n, heads, dim, 3, DTYPES[dtype]), rows(n, heads, dim, 4, DTYPES[dtype])
    slots = torch.arange(n, device="cuda") + 5
    want = expected_pages(np.zeros((2, heads, 16, kv.e8_cache_pages(1, 1, 16, dim).shape[-1]), np.uint32), k, v, slots.tolist(), dim)
    for odd in (1, 3):
        pages = kv.e8_cache_pages(2, heads, 16, dim)
        kv.e8_cache_write(pages, cut_from_wider(k, odd), cut_from_wider(v, odd + 2), slots)
        assert np.array_equal(as_words(pages), want)
    apart = torch.zeros(n * heads * dim * 2 + 1, dtype=DTYPES[dtype], device="cuda")[1:]  # and one that begins at no such multiple either
    apart = apart.as_strided((n, heads, dim), (dim * heads + 1 if n > 1 else 7, dim if heads > 1 else 5, 1))
    apart.copy_(k)
    pages = kv.e8_cache_pages(2, heads, 16, dim)
    kv.e8_cache_write(pages, apart, v.cuda(), slots)
    assert np.array_equal(as_words(pages), want)
    kv.e8_cache_write(pages, rows(21, heads, dim, 5, DTYPES[dtype]).cuda(), rows(21, heads, dim, 6, DTYPES[dtype]).cuda(), torch.arange(21, device="cuda"))
    t, lens = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([21], dtype=torch.int32, device="cuda")
    plainly = kv.e8_cache_attention(k.cuda(), pages, t, lens)
    for odd in (1, 3):
        assert torch.equal(kv.e8_cache_attention(cut_from_wider(k, odd), pages, t, lens), plainly)
    assert torch.equal(kv.e8_cache_attention(apart, pages, t, lens), plainly)
