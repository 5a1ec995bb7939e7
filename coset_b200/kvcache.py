"""E8-coded key/value cache: written as it is quantised, read back, and attended to from the codes.

Beside E8CodeLinear, which keeps a served model's weights as E8 codes, this keeps its keys and values: 4 bits per value and 32 bits per row of
128 values (a row is one token and one head; head_dim is 64, 128 or 256).  A row's step is the smallest bf16 number >= max|x| / 7; its values in
steps are replaced by the nearest point of E8 block by block, f + c / 2 with f a 4-bit number per value and c a bit per block of 8
(the nested pair E8 / 16 Z^8: 32 bits per block as the q = 4, M = 2 code, decoded without a table).  Random keys lose 0.65 dB less than with
whole numbers in the same range.

The cache is paged.  `pages` is int32 [n_pages, n_heads, page_size, words], made by e8_cache_pages; inside a page the layout is the library's
(include/coset_b200.h).  A token's slot is page * page_size + offset; a sequence's row of the page table lists its pages in order.

    pages = e8_cache_pages(n_pages, n_heads, page_size, head_dim)
    e8_cache_write(pages, k, v, slots)                   # k, v [n, n_heads, head_dim] of the new tokens
    y = e8_cache_attention(q, pages, table, lens)        # q [n, q_heads, head_dim]: the last n / len(lens) tokens of every sequence
    k, v = e8_cache_read(pages, slots, torch.bfloat16)   # dense again, for a kernel that wants them so

All of it is for inference: nothing here has a backward pass, and tensors that require gradients are refused outside torch.no_grad().  Calls only
enqueue work on the current stream and may be captured into CUDA graphs.  (No counterpart in the reference.)
"""
from typing import Optional, Tuple, Union

import torch

from . import _lib

_DTYPE_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def e8_cache_pages(n_pages: int, n_heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """An empty cache: every row reads as zeros.  page_size is a power of two from 16 to 1024, head_dim 64, 128 or 256."""
    words = _lib.lib().coset_e8_cache_row_words(int(head_dim))
    if words == 0:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
    if torch.device(device).type != "cuda":
        raise ValueError(f"pages must live on a CUDA device (coset_b200 has no CPU path); got {device}")
    return torch.zeros(n_pages, n_heads, page_size, words, dtype=torch.int32, device=device)


def e8_cache_write(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Quantises keys and values [n, n_heads, head_dim] (float32 or bf16) into the slots (int64 [n]) and returns `pages`.

    Tokens whose slot is negative or behind the last page are left out; the others' slots differ from each other."""
    _lib.native().cache_write(pages, k, v, slots)
    return pages


def e8_cache_read(pages: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of the slots (int64 [n]), each [n, n_heads, head_dim] of dtype float32 or bf16; zeros where a slot is negative
    or behind the last page."""
    return _lib.native().cache_read(pages, slots, _DTYPE_CODES.get(dtype, -1))


def e8_cache_attention(q: torch.Tensor, pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, q_starts: Optional[torch.Tensor] = None,
                       tree: Optional[torch.Tensor] = None, scale: Optional[float] = None, return_lse: bool = False,
                       out: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """softmax(scale * q K^T + mask) V over the cache, for the last tokens of every sequence, which are in the cache already.

    q: [n, q_heads, head_dim] float32 or bf16, the queried tokens of the first sequence, then of the second, ...; q_heads is a multiple of
      the cache's heads, and head h reads cache head h // (q_heads // n_heads).
    table: int32 [n_seqs, max_pages], the pages of each sequence in order; tokens on a page that the cache does not have are not seen.
    lens: int32 [n_seqs], the tokens of each sequence, its queried ones being the last.
    q_starts: int32 [n_seqs + 1], where each sequence's queries begin in q, ascending; by default every sequence has n / n_seqs.
    tree: int64 [n]: bit j of a query's word says whether it sees queried token j of its sequence -- in a tree of drafted tokens its
      ancestors and itself; queried tokens from 64 on are not seen.  By default a query sees the queried tokens up to itself (a chain).  All
      earlier tokens of the sequence are seen.
    scale: 1 / sqrt(head_dim) by default.
    return_lse: also returns log(sum(exp(scale * q K^T + mask))), float32 [n, q_heads], to join the result with attention over other keys.
    out: receives the result (contiguous, of q's shape, type and device, and not q's memory).  Rows of q behind the last sequence are left as
      they were in `out`, and hold anything in a result that is made here.

    A query that sees nothing gives zeros (and -inf).  Queries count with 24 bits from the largest of their row on, sums and the softmax's statistics are
    float32, and weights are rounded to 11 bits for bf16 queries, to 22 for float32 ones.  Where a tree's or a chain's queries of a cache head are
    more than 16 (32 of 64 values) on average over the sequences, bf16 products run on tcgen05 and sum in another order: results agree to the rounding, not
    to the bit.  (A long chain beside many single tokens is faster in a call of its own.)  Equal calls give equal bits.  Of values above 7e31 small
    weights are lost: those below 2^-29 of the largest one there, below 2^-20 at 3e34, 2^-7 at 3e38.

    The call keeps a scratch buffer per device and stream, of 21 MB for heads of 64, 41 MB of 128, 10 MB of 256 (one per call that is captured into a graph, and
    on streams beyond the first 160 of a device)."""
    return _lib.native().cache_attention(q, pages, table, lens, q_starts, tree, None if scale is None else float(scale), bool(return_lse), out)


class E8KVCache:
    """The pages of an E8-coded key/value cache with the calls on them as methods; see the module's functions."""

    def __init__(self, n_pages: int, n_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
        self.pages = e8_cache_pages(n_pages, n_heads, page_size, head_dim, device)
        self.head_dim = head_dim

    @property
    def n_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def n_heads(self) -> int:
        return self.pages.shape[1]

    @property
    def page_size(self) -> int:
        return self.pages.shape[2]

    def write(self, k, v, slots):
        e8_cache_write(self.pages, k, v, slots)

    def read(self, slots, dtype=torch.float32):
        return e8_cache_read(self.pages, slots, dtype)

    def attend(self, q, table, lens, **kw):
        return e8_cache_attention(q, self.pages, table, lens, **kw)
