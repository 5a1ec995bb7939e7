"""The E8-coded key/value cache without a GPU: the plain implementation against a search of its own, refusals of the C ABI and of the Python entry points."""
import ctypes
import itertools
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import kvcache_util as plain


def test_nearest_point_is_the_nearest_of_all_around():
    """Against every point of E8 within one step of the rounded coordinates."""
    g = np.random.RandomState(0)
    u = np.concatenate([g.randint(-28672, 28673, (60, 8)), g.randint(-14, 15, (20, 8)) * 2048, g.randint(-28, 29, (20, 8)) * 1024])
    f, c = plain.nearest(u)
    assert ((f.sum(-1)) % 2 == 0).all() and f.min() >= -8 and f.max() <= 7
    far = ((u - 4096 * f - 2048 * c[:, None]) ** 2).sum(-1)
    steps = np.array(list(itertools.product((-1, 0, 1), repeat=8)))
    for i in range(len(u)):
        for half in (0, 1):
            near = np.floor_divide(u[i] - 2048 * half + 2048, 4096) + steps
            near = near[near.sum(-1) % 2 == 0]
            assert far[i] <= ((u[i] - 4096 * near - 2048 * half) ** 2).sum(-1).min()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_plain_values_follow_from_codes_and_heads(dim):
    x = torch.randn(40, dim, generator=torch.Generator().manual_seed(1))
    codes, heads, v = plain.quantise(x)
    assert torch.equal(plain.values(codes, heads), v)
    step = (heads[:, :1] & np.uint32(0xFFFF0000)).view(np.float32)
    assert (np.abs(x.numpy()).max(-1, keepdims=True) / step <= 7 * (1 + 2.0 ** -22)).all()
    # no point of E8 is further than its covering radius, 1, from anything (and the values were rounded to 1/4096 before)
    off = ((v - x.double()) / torch.from_numpy(step.astype(np.float64))).view(-1, 8).square().sum(-1).sqrt()
    assert float(off.max()) <= 1 + 8 ** 0.5 / 8192 + 1e-5


def _attention(L, **kw):
    a = dict(q=4096, dtype=0, qts=256, qhs=64, n=2, qh=4, pages=4096, n_pages=4, heads=2, page=16, dim=64, table=4096, ts=2, max_pages=2, lens=4096, starts=None,
             seqs=2, tree=None, scale=0.125, out=8192, lse=None, scratch=16384, bytes=1 << 40)
    a.update(kw)
    return L.coset_e8_cache_attention(*a.values(), None)


def test_the_c_abi_refuses_bad_arguments_without_a_gpu():
    """Every call returns before anything is launched: the addresses are made up."""
    from coset_b200 import _lib
    L = _lib.lib()
    assert [L.coset_e8_cache_row_words(d) for d in (64, 128, 256)] == [18, 34, 68]
    assert [L.coset_e8_cache_row_words(d) for d in (0, 8, 96, 512, -1)] == [0] * 5
    assert L.coset_e8_cache_attention_scratch_bytes(128) > 0 and L.coset_e8_cache_attention_scratch_bytes(100) == 0

    def write(pages=4096, n_pages=4, heads=2, page=16, dim=64, k=4096, kt=128, kh=64, v=4096, vt=128, vh=64, dtype=0, slots=4096, n=3):
        return L.coset_e8_cache_write(pages, n_pages, heads, page, dim, k, kt, kh, v, vt, vh, dtype, slots, n, None)

    def read(pages=4096, n_pages=4, heads=2, page=16, dim=64, slots=4096, n=3, k=4096, v=8192, dtype=0):
        return L.coset_e8_cache_read(pages, n_pages, heads, page, dim, slots, n, k, v, dtype, None)

    for call in (write, read, lambda **kw: _attention(L, **kw)):
        for kw in (dict(dim=96), dict(dim=0), dict(page=8), dict(page=24), dict(page=2048), dict(page=0), dict(page=-16), dict(heads=0), dict(heads=70000),
                   dict(n_pages=-1), dict(n_pages=1 << 31), dict(pages=None), dict(pages=4100), dict(n=-1), dict(dtype=2), dict(dtype=-1)):
            assert call(**kw) < 0, kw
            assert L.coset_last_error_string()
        assert call(n=0) == 0
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(k=4100), dict(v=4104), dict(slots=4100), dict(kt=127), dict(kh=2), dict(vt=6, dtype=0), dict(vh=4, dtype=1),
               dict(n=1 << 62), dict(n=1 << 40)):
        assert write(**kw) < 0, kw
    for kw in (dict(k=None), dict(v=None), dict(slots=None), dict(k=4100), dict(v=4104), dict(slots=4100), dict(n=1 << 62), dict(n=1 << 40)):
        assert read(**kw) < 0, kw
    for kw in (dict(q=None), dict(q=4100), dict(out=None), dict(out=8200), dict(qts=2), dict(qhs=7), dict(qh=3), dict(qh=0), dict(lens=None), dict(table=None), dict(max_pages=-1),
               dict(seqs=-1), dict(seqs=0), dict(n=3), dict(scratch=None), dict(bytes=0), dict(scratch=16392), dict(max_pages=1 << 30), dict(ts=-1)):
        assert _attention(L, **kw) < 0, kw
        assert L.coset_last_error_string()


def test_tensors_off_the_gpu_are_refused():
    from coset_b200 import kvcache as kv
    pages, x, s = torch.zeros(1, 2, 16, 18, dtype=torch.int32), torch.zeros(2, 2, 64), torch.arange(2)
    with pytest.raises(ValueError, match="CUDA"):
        kv.e8_cache_pages(1, 2, 16, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        kv.e8_cache_write(pages, x, x, s)
    with pytest.raises(ValueError, match="CUDA"):
        kv.e8_cache_read(pages, s)
    with pytest.raises(ValueError, match="CUDA"):
        kv.e8_cache_attention(x, pages, s.int().view(2, 1), s.int())
    for dim, page in ((80, 16), (64, 24), (64, 8), (64, 2048)):
        with pytest.raises(ValueError):
            kv.e8_cache_pages(1, 2, page, dim)
