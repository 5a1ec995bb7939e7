"""The E8-coded key/value cache on the GPU: pages to the bit, values, and attention against 64 bits."""
import math
import os
import random
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import kvcache_util as plain

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def api():
    from coset_b200 import kvcache
    return kvcache


def rows(n, heads, dim, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, dim, generator=g) * torch.exp(0.5 * torch.randn(1, heads, dim, generator=g))
    return x.to(dtype)


def special_rows(dim, dtype):
    """Rows at which a quantiser can go wrong: [n, dim]."""
    inf, nan = math.inf, math.nan
    x = torch.zeros(24, dim)
    x[1] = 1e-35                                          # below the smallest row that is kept
    x[2] = 2.0 ** -100
    x[3] = 2.0 ** -99.9
    x[4, dim - 1] = 3.3e38
    x[5] = 7.0
    x[6] = -7.0
    x[7] = torch.randint(-7, 8, (dim,), generator=torch.Generator().manual_seed(1)).float()        # points of Z^8: ties of the moved coordinate
    x[7, 0] = 7.0
    x[8] = torch.randint(-14, 15, (dim,), generator=torch.Generator().manual_seed(2)).float() / 2  # halves: ties of the rounding
    x[8, 0] = 7.0
    x[9] = torch.randint(-28, 29, (dim,), generator=torch.Generator().manual_seed(3)).float() / 4  # quarters: ties between the cosets
    x[9, 1] = -7.0
    x[10] = 0.5
    x[10, 3] = 7.0
    x[11] = torch.arange(dim) * 1e-3
    x[12, 2] = inf
    x[13, 5] = -inf
    x[14, 0] = nan
    x[15] = nan
    x[16, 0], x[16, 1] = nan, inf
    x[17] = 1e-3
    x[17, dim // 2] = 1e3                                 # one outlier
    x[18, 9] = -1e-45 if dtype == torch.float32 else -1e-40
    x[19] = (torch.arange(dim) % 3 - 1) * 3e38
    x[20] = 6.99999
    x[20, ::2] = -3.4999
    x[21, 8:16] = 1.0
    x[22] = torch.randn(dim, generator=torch.Generator().manual_seed(4)) * 1e-30
    x[23] = torch.randn(dim, generator=torch.Generator().manual_seed(5)) * 1e30
    return x.to(dtype)


def expected_pages(before, k, v, slots, dim):
    want = before.copy()
    kc, kh, vc, vh = plain.planes(want, dim)
    P, H, S, _ = want.shape
    for x, codes, heads in ((k, kc, kh), (v, vc, vh)):
        for t, slot in enumerate(slots):
            if 0 <= slot < P * S:
                c, h, _ = plain.quantise(x[t])
                codes[slot // S, :, slot % S], heads[slot // S, :, slot % S] = c, h
    return want


def as_words(pages):
    return pages.cpu().numpy().view(np.uint32)


# ------------------------------------------------------------------ writing
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim, heads, page, n", [(64, 1, 16, 1), (64, 12, 16, 37), (128, 8, 64, 70), (128, 3, 32, 1), (256, 2, 128, 33), (256, 1, 1024, 5)])
def test_written_pages_are_the_definition_to_the_bit(dtype, dim, heads, page, n):
    kv = api()
    n_pages = (n + page - 1) // page + 2
    k, v = rows(n, heads, dim, 1, DTYPES[dtype]), rows(n, heads, dim, 2, DTYPES[dtype])
    slots = random.Random(n).sample(range(n_pages * page), n)
    if n > 3:
        slots[2], slots[3] = -1, n_pages * page  # neither is written
    pages = kv.e8_cache_pages(n_pages, heads, page, dim)
    before = torch.randint(-2 ** 31, 2 ** 31, pages.shape, dtype=torch.int64, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    pages.copy_(before)
    version = pages._version
    got = kv.e8_cache_write(pages, k.cuda(), v.cuda(), torch.tensor(slots, device="cuda"))
    assert got is pages and pages._version > version
    want = expected_pages(before.numpy().view(np.uint32), k, v, slots, dim)
    assert np.array_equal(as_words(pages), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_special_rows(dtype, dim):
    kv = api()
    x = special_rows(dim, DTYPES[dtype])
    n = len(x)
    k, v = x.view(n, 1, dim), x.flip(0).reshape(n, 1, dim)
    pages = kv.e8_cache_pages(2, 1, 16, dim)
    slots = list(range(n))
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), torch.tensor(slots, device="cuda"))
    assert np.array_equal(as_words(pages), expected_pages(np.zeros(pages.shape, np.uint32), k, v, slots, dim))
    got = kv.e8_cache_read(pages, torch.tensor(slots, device="cuda"), torch.float32)
    want = plain.quantise(x)[2].float()
    assert torch.equal(torch.nan_to_num(got[0].cpu().view(n, dim), nan=1.5), torch.nan_to_num(want, nan=1.5))
    assert torch.isnan(got[0][12:17]).all()


def test_many_random_blocks_and_ties():
    """A million blocks, a quarter of them on grids full of ties, against the plain search."""
    kv = api()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(65536, 128, generator=g)
    x[:8192] = torch.randint(-14, 15, (8192, 128), generator=g).float() / 2
    x[8192:16384] = torch.randint(-56, 57, (8192, 128), generator=g).float() / 8
    x[:16384, 0] = 7.0
    pages = kv.e8_cache_pages(1024, 1, 64, 128)
    slots = torch.arange(65536, device="cuda")
    kv.e8_cache_write(pages, x.view(-1, 1, 128).cuda(), x.bfloat16().float().view(-1, 1, 128).cuda(), slots)
    kc, kh, vc, vh = plain.planes(as_words(pages), 128)
    for codes, heads, y in ((kc, kh, x), (vc, vh, x.bfloat16().float())):
        c, h, _ = plain.quantise(y)
        assert np.array_equal(codes.reshape(c.shape), c) and np.array_equal(heads.reshape(h.shape), h)


def test_strides_alignment_and_other_orders():
    """Keys and values as views of one projection, heads first, not aligned, broadcast over heads."""
    kv = api()
    n, heads, dim, page = 21, 4, 64, 16
    wide = rows(n, 3 * heads, dim, 5)
    slots = torch.randperm(48, generator=torch.Generator().manual_seed(1))[:n]
    cases = [(wide.cuda()[:, heads:2 * heads], wide.cuda()[:, 2 * heads:], wide[:, heads:2 * heads], wide[:, 2 * heads:])]
    first = wide.transpose(0, 1).contiguous().cuda()  # [heads, n, dim]
    cases.append((first[:heads].transpose(0, 1), first[heads:2 * heads].transpose(0, 1), wide[:, :heads], wide[:, heads:2 * heads]))
    flat = torch.zeros(n * heads * dim + 1, device="cuda")
    flat[1:] = wide[:, :heads].reshape(-1).cuda()
    off = flat[1:].view(n, heads, dim)
    assert off.data_ptr() % 16
    cases.append((off, off, wide[:, :heads], wide[:, :heads]))
    one = wide[:, :1].cuda().expand(n, heads, dim)
    cases.append((one, one, wide[:, :1].expand(n, heads, dim), wide[:, :1].expand(n, heads, dim)))
    last = wide[:, :heads].transpose(1, 2).contiguous().cuda().transpose(1, 2)  # values of a row are not neighbours
    cases.append((last, last, wide[:, :heads], wide[:, :heads]))
    for k, v, kw, vw in cases:
        pages = kv.e8_cache_pages(3, heads, page, dim)
        kv.e8_cache_write(pages, k, v, slots.cuda())
        assert np.array_equal(as_words(pages), expected_pages(np.zeros(pages.shape, np.uint32), kw, vw, slots.tolist(), dim))
        spread = torch.stack([slots, slots], 1).cuda()[:, 0]  # slots with a stride
        assert torch.equal(kv.e8_cache_read(pages, spread)[0], kv.e8_cache_read(pages, slots.cuda())[0])


def test_nothing_to_write_or_read():
    kv = api()
    pages = kv.e8_cache_pages(1, 2, 16, 64)
    none = torch.empty(0, 2, 64, device="cuda")
    kv.e8_cache_write(pages, none, none, torch.empty(0, dtype=torch.int64, device="cuda"))
    k, v = kv.e8_cache_read(pages, torch.empty(0, dtype=torch.int64, device="cuda"), torch.bfloat16)
    assert k.shape == v.shape == (0, 2, 64) and k.dtype == torch.bfloat16
    empty = kv.e8_cache_pages(0, 2, 16, 64)  # a cache without pages: every slot is outside it
    kv.e8_cache_write(empty, torch.ones(3, 2, 64, device="cuda"), torch.ones(3, 2, 64, device="cuda"), torch.arange(3, device="cuda"))
    assert not kv.e8_cache_read(empty, torch.arange(3, device="cuda"))[0].any()


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim, heads, page", [(64, 12, 16), (128, 8, 64), (256, 3, 32)])
def test_read_back(dtype, dim, heads, page):
    kv = api()
    pages = kv.e8_cache_pages(5, heads, page, dim)
    k, v = rows(5 * page, heads, dim, 8), rows(5 * page, heads, dim, 9)
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), torch.arange(5 * page, device="cuda"))
    slots = [3, 3, 5 * page - 1, -1, 0, 5 * page, 2 ** 40, -2 ** 62, page] + list(range(7, 40))  # a slot may be read twice
    got = kv.e8_cache_read(pages, torch.tensor(slots, device="cuda"), DTYPES[dtype])
    for x, y in zip((k, v), got):
        for t, slot in enumerate(slots):
            want = plain.quantise(x[slot])[2] if 0 <= slot < 5 * page else torch.zeros(heads, dim)
            assert torch.equal(y[t].cpu(), want.to(DTYPES[dtype])), (t, slot)


def test_offsets_beyond_32_bits():
    """Pages whose words, and bytes, 32 bits cannot count: 2^31 words are 8 GB."""
    kv = api()
    heads, page, dim = 8, 1024, 128
    n_pages = 2 ** 31 // (heads * page * 34) + 3
    pages = kv.e8_cache_pages(n_pages, heads, page, dim)
    k, v = rows(20, heads, dim, 11, torch.bfloat16), rows(20, heads, dim, 12, torch.bfloat16)
    slots = torch.tensor([n_pages * page - 1 - 5 * i for i in range(19)] + [7])
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), slots.cuda())
    got = kv.e8_cache_read(pages, slots.cuda(), torch.float32)
    for x, y in zip((k, v), got):
        assert torch.equal(y.cpu().view(-1, dim), plain.quantise(x.reshape(-1, dim))[2].float())
    table = torch.tensor([[n_pages - 1, 0]], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, heads, dim, device="cuda")
    y = kv.e8_cache_attention(q, pages, table, torch.tensor([page + 8], dtype=torch.int32, device="cuda"))
    vs = torch.cat([kv.e8_cache_read(pages, torch.arange(page, device="cuda") + (n_pages - 1) * page)[1], kv.e8_cache_read(pages, torch.arange(8, device="cuda"))[1]])
    assert torch.allclose(y[0], vs.double().mean(0).float(), rtol=0, atol=2.0 ** -19 * float(vs.abs().mean(0).max()))
    del pages
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ attention
def filled(dim, heads, page, lens, seed, dtype=torch.bfloat16, spare=2):
    """A cache with sequences of these lengths, their pages in any order, and its page table; rows that no sequence uses are full of numbers."""
    kv = api()
    r = random.Random(seed)
    need = [(n + page - 1) // page for n in lens]
    n_pages = sum(need) + spare
    pages = kv.e8_cache_pages(n_pages, heads, page, dim)
    k, v = rows(n_pages * page, heads, dim, seed, dtype), rows(n_pages * page, heads, dim, seed + 1, dtype)
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), torch.arange(n_pages * page, device="cuda"))
    order = r.sample(range(n_pages), sum(need))
    table, at = [], 0
    for m in need:
        table.append(order[at:at + m] + [0] * (max(need + [1]) - m))
        at += m
    return pages, table


def random_tree(counts, seed):
    r, words = random.Random(seed), []
    for n in counts:
        seen = []
        for j in range(n):
            up = r.randrange(-1, j)
            seen.append((seen[up] if up >= 0 else 0) | 1 << j)
        words += seen
    return words


def signed(words):
    return torch.tensor([w - (1 << 64) if w >> 63 else w for w in words], dtype=torch.int64, device="cuda")


def check(q, pages, dim, table, lens, starts, tree, scale=None, got=None, **kw):
    """Compares with 64 bits.

    Errors that are counted: a score is a float32 sum of dim (and dim / 8) products of q, kept to 2^-22, with whole numbers up to 31/2, twice the
    largest coordinate of a point -- so at most (2^-22 + (dim + 32) 2^-24) reach * 4, relative to a weight, or for random signs a tenth of that; four
    roundings (scale, subtraction, exp2 to 2^-22, its argument) more.  A weight is rounded to 2^-12 for bf16 queries, to 2^-22 for float32, and its
    sums with whole numbers are float32.  The result is rounded once."""
    kv = api()
    scale = 1 / math.sqrt(dim) if scale is None else scale
    if got is None:
        got = kv.e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                    q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), tree=None if tree is None else signed(tree),
                                    scale=scale, return_lse=True, **kw)
    out, lse, spread, reach = plain.attend(q.cpu().double(), as_words(pages), dim, table, lens, starts, tree, scale)
    y, z = got[0].cpu().double(), got[1].cpu().double()
    assert y.shape == q.shape and got[0].dtype == q.dtype and got[1].dtype == torch.float32
    live = starts[-1]
    y, z, out, lse, spread, reach = (t[:live] for t in (y, z, out, lse, spread, reach))
    score = (2.0 ** -22 + (dim + 32) * 2.0 ** -24) * 4 * reach + 2.0 ** -20
    weight = 2.0 ** -12 if q.dtype == torch.bfloat16 else 2.0 ** -22
    bound = torch.finfo(q.dtype).eps / 2 * out.abs() + (2 * score + 2 * weight + 2.0 ** -18) * spread + 1e-30
    worst = (y - out).abs() / bound
    at, most = np.unravel_index(int(worst.argmax()), worst.shape), float(worst.max())
    assert most <= 1.0, f"out: {most} of the bound at {at}"  # not a number fails too
    none = lse == -math.inf
    assert torch.equal(z == -math.inf, none)
    far = ((z - lse).abs() / (score.squeeze(-1) + 2.0 ** -22 * lse.abs()))[~none]
    most = float(far.max()) if far.numel() else 0.0
    assert most <= 1.0, f"lse: {most} of the bound"
    return got


def starts_of(counts):
    return [0] + np.cumsum(counts).tolist()


SHAPES = [
    # dim, heads, group, page, lens, queried tokens
    (64, 1, 1, 16, [1], [1]),
    (128, 1, 4, 16, [2, 1, 33], [1, 1, 1]),
    (128, 2, 4, 64, [64, 63, 65, 128, 127, 1], [1] * 6),
    (64, 12, 1, 16, [100, 257, 512], [1] * 3),
    (256, 2, 2, 32, [31, 300], [1, 1]),
    (128, 1, 8, 64, [700], [1]),
    (128, 2, 7, 32, [90, 200], [1, 1]),            # seven query heads per head
    (128, 1, 16, 128, [130, 400], [1, 1]),
    (128, 2, 4, 64, [300, 64, 65], [4, 4, 4]),
    (64, 2, 3, 16, [50, 20], [5, 5]),
    (256, 1, 4, 64, [150, 77], [6, 6]),
    (128, 1, 4, 64, [333], [64]),
    (64, 1, 8, 32, [100, 70], [64, 64]),
    (256, 1, 5, 32, [200], [33]),
    (128, 2, 1, 64, [200], [17]),
]


@pytest.mark.parametrize("mask", ["chain", "tree"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"d{s[0]}h{s[1]}g{s[2]}p{s[3]}n{max(s[4])}t{max(s[5])}")
def test_attention(shape, dtype, mask):
    dim, heads, group, page, lens, counts = shape
    pages, table = filled(dim, heads, page, lens, 7)
    q = (rows(sum(counts), heads * group, dim, 21) * 1.5).to(DTYPES[dtype]).cuda()
    tree = random_tree(counts, 3) if mask == "tree" else None
    got = check(q, pages, dim, table, lens, starts_of(counts), tree)
    if len(set(counts)) == 1:  # the same without saying where the queries begin
        kv = api()
        again = kv.e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                      tree=None if tree is None else signed(tree), return_lse=True)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])  # and the same bits every time


MANY_ROWS = [
    # rows of a cache head (group x queried tokens) around the sizes of tiles, lengths around theirs, segments that many CTAs share
    (128, 1, 16, 16, [40], [1]),
    (128, 1, 17, 16, [40], [1]),
    (128, 1, 128, 16, [1], [1]),
    (128, 2, 4, 16, [129, 128, 127], [5, 5, 5]),
    (64, 1, 32, 32, [300], [1]),
    (64, 1, 11, 32, [257], [3]),
    (128, 1, 4, 64, [500, 37], [32, 32]),
    (128, 1, 4, 64, [500, 37], [33, 33]),
    (64, 2, 5, 1024, [1500], [51]),
    (64, 1, 4, 16, [1000], [64]),
    (128, 1, 6, 16, [900], [50]),
    (64, 1, 8, 16, [2000], [64]),
    (128, 1, 4, 128, [20000], [16]),
    (128, 1, 8, 64, [9000, 9], [40, 40]),
    (64, 2, 8, 64, [10000], [20]),
]


@pytest.mark.parametrize("mask", ["chain", "tree"])
@pytest.mark.parametrize("shape", MANY_ROWS, ids=lambda s: f"d{s[0]}h{s[1]}g{s[2]}p{s[3]}n{max(s[4])}t{max(s[5])}")
def test_attention_of_many_rows(shape, mask):
    dim, heads, group, page, lens, counts = shape
    pages, table = filled(dim, heads, page, lens, 17)
    q = (rows(sum(counts), heads * group, dim, 22) * 1.5).to(torch.bfloat16).cuda()
    check(q, pages, dim, table, lens, starts_of(counts), random_tree(counts, 5) if mask == "tree" else None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim, group, lens, count", [(64, 2, [250, 190], 190), (128, 4, [300], 100), (256, 1, [140], 140)])
def test_chains_longer_than_a_tree_can_be(dim, group, lens, count, dtype):
    pages, table = filled(dim, 1, 16, lens, 18)
    q = rows(count * len(lens), group, dim, 23, DTYPES[dtype]).cuda()
    check(q, pages, dim, table, lens, starts_of([count] * len(lens)), None)


@pytest.mark.parametrize("dim", [64, 128])
def test_many_rows_in_a_ragged_batch(dim):
    """Sequences without queries, without tokens, with more queries than tokens, some of one tile and some of two; rows behind the last stay."""
    lens, counts = [70, 0, 3, 400, 0, 129, 5], [64, 2, 9, 60, 0, 40, 1]
    pages, table = filled(dim, 2, 32, lens, 4)
    starts = starts_of(counts)
    q = rows(starts[-1] + 4, 10, dim, 5, torch.bfloat16).cuda()
    for tree in (None, random_tree(counts, 8) + [0] * 4):
        out = torch.full_like(q, 5.0)
        check(q, pages, dim, table, lens, starts, tree, out=out)
        assert (out[starts[-1]:] == 5.0).all()


@pytest.mark.parametrize("most", [2, 14])
@pytest.mark.parametrize("n", [33, 70])
def test_more_sequences_than_a_warp_has_lanes(n, most):
    r = random.Random(n + most)
    lens, counts = [r.randrange(0, 150) for _ in range(n)], [r.randrange(0, most + 1) for _ in range(n)]
    pages, table = filled(128, 1, 16, lens, 6)
    q = rows(sum(counts), 4, 128, 7, torch.bfloat16).cuda()
    check(q, pages, 128, table, lens, starts_of(counts), None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_ragged_batch_with_empty_sequences_and_rows_behind_the_last(dim, dtype):
    """Sequences without queries, without tokens, with more queries than tokens; rows behind the last sequence stay."""
    kv = api()
    lens, counts = [70, 0, 3, 200, 0, 129, 5], [3, 2, 5, 0, 0, 20, 1]
    pages, table = filled(dim, 2, 32, lens, 4)
    starts = starts_of(counts)
    q = rows(starts[-1] + 4, 6, dim, 5, DTYPES[dtype]).cuda()
    for tree in (None, random_tree(counts, 8) + [0] * 4):
        out = torch.full_like(q, 5.0)
        got = check(q, pages, dim, table, lens, starts, tree, out=out)
        assert got[0] is out or got[0].data_ptr() == out.data_ptr()
        assert (out[starts[-1]:] == 5.0).all()


@pytest.mark.parametrize("tokens", [1, 12])
def test_long_sequences_split_over_the_chip(tokens):
    """A sequence that many CTAs share, beside short ones."""
    dim, lens = 128, [5000, 3, 40]
    pages, table = filled(dim, 1, 64, lens, 9)
    counts = [tokens] * 3
    q = rows(3 * tokens, 4, dim, 2, torch.bfloat16).cuda()
    check(q, pages, dim, table, lens, starts_of(counts), None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens", [2, 12, 40])
def test_masked_places_hold_anything(tokens, dtype):
    """Infinities and NaN in tokens that a query does not see, and behind a sequence's end, leave its result alone; what it sees they reach."""
    kv = api()
    dim, heads, page = 128, 1, 16
    L = 60
    pages, table = filled(dim, heads, page, [L], 3)
    slot = lambda i: table[0][i // page] * page + i % page  # noqa: E731
    bad_at = [L - tokens + 1, L, L + 1, L + 2]  # queried token 1, and the rest of the last page
    assert (L + 2) // page == (L - 1) // page
    bad = torch.zeros(4, heads, dim)
    bad[0, 0, 3], bad[1, 0, 0], bad[2, 0, 5], bad[3] = math.nan, math.inf, -math.inf, 3e38
    at = torch.tensor([slot(i) for i in bad_at], device="cuda")
    kv.e8_cache_write(pages, bad.cuda(), bad.flip(0).cuda(), at)
    tree = [1 << i | 1 if i != 1 else 2 for i in range(tokens)]  # all see token 0 and themselves; token 1 sees itself alone
    q = rows(tokens, 4, dim, 6, DTYPES[dtype]).cuda()
    args = (q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([L], dtype=torch.int32, device="cuda"))
    y, z = kv.e8_cache_attention(*args, tree=signed(tree), return_lse=True)
    assert torch.isnan(y[1]).all() and torch.isnan(z[1]).all()
    others = [i for i in range(tokens) if i != 1]
    clean = as_words(pages).copy()
    for p in plain.planes(clean, dim):
        p[slot(L - tokens + 1) // page, :, slot(L - tokens + 1) % page] = 0
    want = plain.attend(q.cpu().double(), clean, dim, table, [L], [0, tokens], tree, 1 / math.sqrt(dim))
    assert torch.allclose(y[others].cpu().double(), want[0][others], rtol=2.0 ** -7, atol=2.0 ** -9) and torch.isfinite(y[others]).all()


@pytest.mark.parametrize("dtype, group", [("f32", 2), ("bf16", 2), ("bf16", 24), ("bf16", 72)])
def test_values_of_very_different_sizes(dtype, group):
    """Values from 1e-30 to 1e30 in one sequence, rows of zeros, a huge value that one query does not see; scores that overflow exp."""
    kv = api()
    dim, page, L = 64, 16, 80
    pages, table = filled(dim, 1, page, [L], 3)
    slots = torch.tensor([table[0][i // page] * page + i % page for i in range(L)], device="cuda")
    k, v = rows(L, 1, dim, 30), rows(L, 1, dim, 31)
    v *= torch.tensor([10.0 ** (i % 13 - 6) for i in range(L)]).view(L, 1, 1)
    v[10:14], k[20:24] = 0, 0
    v[-1] = 1e30
    k[5] *= 40
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), slots)
    q = (rows(2, group, dim, 32) * 6).to(DTYPES[dtype]).cuda()
    check(q, pages, dim, table, [L], [0, 2], [1, 2])  # the first of two queried tokens does not see the last
    v[:] = 0
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), slots)
    y = kv.e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([L], dtype=torch.int32, device="cuda"))
    assert float(y.abs().max()) <= 1e-25
    v = rows(L, 1, dim, 33) * 1e-30
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), slots)
    if dtype == "f32":
        check(q, pages, dim, table, [L], [0, 2], None)


@pytest.mark.parametrize("group", [2, 20])
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 300.0, 1e30])
def test_queries_of_every_size(size, group):
    dim = 128
    pages, table = filled(dim, 1, 16, [50], 13)
    q = rows(3, group, dim, 14) * size
    q[0, 0, 5] = 50 * size
    q[1, 1] = 0
    for dtype in (torch.float32, torch.bfloat16):
        check(q.to(dtype).cuda(), pages, dim, table, [50], [0, 3], None, scale=min(1.0, 1.0 / size) / math.sqrt(dim))


@pytest.mark.parametrize("group, dtype", [(1, "f32"), (24, "bf16"), (80, "bf16")])
def test_pages_outside_the_cache_are_not_seen(group, dtype):
    kv = api()
    dim, page = 64, 16
    lens = [60, 40]
    pages, table = filled(dim, 2, page, lens, 5)
    table[0][1], table[1][0], table[1][1], table[1][2] = -1, pages.shape[0], 2 ** 31 - 1, -2 ** 31
    q = rows(4, 2 * group, dim, 6, DTYPES[dtype]).cuda()
    got = check(q, pages, dim, table, lens, [0, 2, 4], None)
    assert torch.equal(got[0][2:], torch.zeros_like(got[0][2:])) and (got[1][2:] == -math.inf).all()
    lens = [1000, 100]  # more than the table lists
    table = [table[0], [0, 1, 2, 3]]
    check(q, pages, dim, table, [min(n, 64) for n in lens], [0, 2, 4], None,
          got=kv.e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True))
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    y, z = kv.e8_cache_attention(q, pages, none, torch.tensor(lens, dtype=torch.int32, device="cuda"), return_lse=True)
    assert not y.any() and (z == -math.inf).all()
    y, z = kv.e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([-5, -2 ** 31], dtype=torch.int32, device="cuda"), return_lse=True)
    assert not y.any() and (z == -math.inf).all()


@pytest.mark.parametrize("heads, dtype", [(2, torch.float32), (24, torch.bfloat16), (80, torch.bfloat16)])
def test_starts_that_make_no_sense_touch_nothing_outside(heads, dtype):
    """Starts that descend, lie outside, or overlap: every access stays inside, and a later call is right."""
    kv = api()
    pages, table = filled(64, 1, 16, [40, 40, 40], 5)
    q = rows(6, heads, 64, 6, dtype).cuda()
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([40] * 3, dtype=torch.int32, device="cuda")
    for starts in ([0, 4, 2, 6], [-5, 2, 100, 2 ** 31 - 1], [-2 ** 31, -1, -1, 3], [6, 6, 6, 6], [0, 2 ** 31 - 1, 0, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31]):
        guard = torch.full((18, heads, 64), 3.0, dtype=dtype, device="cuda")
        kv.e8_cache_attention(q, pages, t, n, q_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=guard[6:12])
        assert (guard[:6] == 3.0).all() and (guard[12:] == 3.0).all()
    check(q, pages, 64, table, [40] * 3, [0, 1, 3, 6], None)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("dim, group, dtype", [(64, 2, "f32"), (128, 2, "bf16"), (128, 24, "bf16"), (64, 70, "bf16")])
def test_scales(dim, group, dtype, scale):
    pages, table = filled(dim, 1, 16, [70, 33], 8)
    q = rows(4, group, dim, 9, DTYPES[dtype]).cuda()
    check(q, pages, dim, table, [70, 33], [0, 2, 4], None, scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_broadcast_rows_and_parts_of_a_cache(dtype):
    """Keys that all heads share are written from one copy; the pages from some page on are a cache of their own."""
    kv = api()
    dim, page = 128, 16
    whole = kv.e8_cache_pages(5, 3, page, dim)
    k, v = rows(20, 1, dim, 1, DTYPES[dtype]).cuda(), rows(20, 3, dim, 2, DTYPES[dtype]).cuda()
    slots = torch.arange(20, device="cuda")
    part = whole[2:]
    kv.e8_cache_write(part, k.expand(20, 3, dim), v, slots)
    other = kv.e8_cache_pages(3, 3, page, dim)
    kv.e8_cache_write(other, k.expand(20, 3, dim).contiguous(), v, slots)
    assert torch.equal(part, other) and not whole[:2].any()
    q = rows(1, 6, dim, 3, DTYPES[dtype]).cuda()
    t, n = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    assert torch.equal(kv.e8_cache_attention(q, part, t, n), kv.e8_cache_attention(q, whole, t + 2, n))


def test_queries_in_other_orders_and_no_queries():
    kv = api()
    dim, lens = 128, [77, 20]
    pages, table = filled(dim, 2, 16, lens, 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = rows(4, 24, dim, 3, torch.bfloat16).cuda()
    plainly = kv.e8_cache_attention(wide[:, 8:16].contiguous(), pages, t, n)
    assert torch.equal(plainly, kv.e8_cache_attention(wide[:, 8:16], pages, t, n))
    first = wide[:, 8:16].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(plainly, kv.e8_cache_attention(first, pages, t, n))
    off = torch.zeros(4 * 8 * dim + 1, dtype=torch.bfloat16, device="cuda")
    off[1:] = wide[:, 8:16].reshape(-1)
    assert torch.equal(plainly, kv.e8_cache_attention(off[1:].view(4, 8, dim), pages, t, n))
    wider = torch.full((2, t.shape[1] + 3), 2 ** 31 - 1, dtype=torch.int32, device="cuda")  # rows of a larger table
    wider[:, :t.shape[1]] = t
    assert torch.equal(plainly, kv.e8_cache_attention(wide[:, 8:16], pages, wider[:, :t.shape[1]], n))
    assert torch.equal(plainly, kv.e8_cache_attention(wide[:, 8:16], pages, t.T.contiguous().T, n))
    y, z = kv.e8_cache_attention(wide[:0, :8], pages, t, n, return_lse=True)
    assert y.shape == (0, 8, dim) and z.shape == (0, 8)
    y = kv.e8_cache_attention(wide[:0, :8], pages, t[:0], n[:0])
    assert y.shape == (0, 8, dim)


# ------------------------------------------------------------------ the calls as a serving program makes them
def test_generation_step_by_step_in_a_graph():
    """Prompt, then steps of write and attend captured once and replayed while the cache and the lengths grow; two graphs and an eager call on
    another stream between them."""
    kv = api()
    dim, heads, group, page, B = 128, 2, 4, 16, 3
    cache = kv.E8KVCache(12, heads, dim, page)
    table = [[0, 5, 7, 9], [1, 2, 3, 11], [4, 6, 8, 10]]
    t = torch.tensor(table, dtype=torch.int32, device="cuda")
    prompt = [20, 15, 33]
    slots = torch.tensor([table[b][i // page] * page + i % page for b in range(B) for i in range(prompt[b])], device="cuda")
    k, v = rows(sum(prompt), heads, dim, 1, torch.bfloat16).cuda(), rows(sum(prompt), heads, dim, 2, torch.bfloat16).cuda()
    cache.write(k, v, slots)
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    place = torch.zeros(B, dtype=torch.int64, device="cuda")
    q, kn, vn = (torch.zeros(B, h, dim, dtype=torch.bfloat16, device="cuda") for h in (heads * group, heads, heads))

    def step():
        cache.write(kn, vn, place)
        return cache.attend(q, t, lens, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        place.fill_(-1)
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(step())
    now = list(prompt)
    for i in range(14):
        new = [rows(B, h, dim, 50 + 3 * i + j, torch.bfloat16) for j, h in enumerate((heads * group, heads, heads))]
        for dst, src in zip((q, kn, vn), new):
            dst.copy_(src)
        place.copy_(torch.tensor([table[b][now[b] // page] * page + now[b] % page for b in range(B)]))
        now = [x + 1 for x in now]
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        if i % 3 == 2:
            with torch.cuda.stream(side):
                other = cache.attend(q.clone(), t, lens)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        check(q, cache.pages, dim, table, now, list(range(B + 1)), None, got=results[i % 2])


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_two_captured_graphs_at_once(tokens):
    """Two graphs of the same call replayed on two streams at the same time, with lengths that changed since, beside eager calls."""
    kv = api()
    dim = 128
    pages, table = filled(dim, 2, 16, [900, 300], 5)
    t = torch.tensor(table, dtype=torch.int32, device="cuda")
    tree = signed(random_tree([tokens] * 2, 9))
    lens = torch.tensor([100, 60], dtype=torch.int32, device="cuda")
    q = rows(2 * tokens, 8, dim, 3, torch.bfloat16).cuda()
    kv.e8_cache_attention(q, pages, t, lens, tree=tree)
    streams, graphs, results = [torch.cuda.Stream() for _ in range(2)], [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(kv.e8_cache_attention(q, pages, t, lens, tree=tree))
    for now in ([900, 300], [64, 64], [577, 1]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(10):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            want = kv.e8_cache_attention(q, pages, t, lens, tree=tree)
        torch.cuda.synchronize()
        assert torch.equal(results[0], want) and torch.equal(results[1], want)


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_two_streams_and_two_threads_at_once(tokens):
    import threading
    kv = api()
    dim = 128
    pages, table = filled(dim, 2, 16, [900, 300], 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([900, 300], dtype=torch.int32, device="cuda")
    qs = [rows(2 * tokens, 8, dim, s, torch.bfloat16).cuda() for s in range(4)]
    want = [kv.e8_cache_attention(q, pages, t, n) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(kv.e8_cache_attention(qs[i], pages, t, n), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not wrong


def test_a_run_of_the_operators_together():
    """Prompt, a tree of drafted tokens verified, the accepted ones kept, the cache read back and attended to densely: all three agree."""
    kv = api()
    dim, heads, group, page = 64, 2, 2, 16
    cache = kv.E8KVCache(8, heads, dim, page)
    table = [[3, 0, 6, 2]]
    at = lambda i: table[0][i // page] * page + i % page  # noqa: E731
    ctx, drafted = 21, 6
    k, v = rows(ctx + drafted, heads, dim, 1), rows(ctx + drafted, heads, dim, 2)
    slots = torch.tensor([at(i) for i in range(ctx + drafted)], device="cuda")
    cache.write(k[:ctx].cuda(), v[:ctx].cuda(), slots[:ctx])
    cache.write(k[ctx:].cuda(), v[ctx:].cuda(), slots[ctx:])
    tree = [0b000001, 0b000011, 0b000101, 0b001011, 0b010101, 0b100000]
    q = rows(drafted, heads * group, dim, 3).cuda()
    y, z = check(q, cache.pages, dim, table, [ctx + drafted], [0, drafted], tree)
    kd, vd = cache.read(slots, torch.float32)
    # the path 0, 1, 3 is accepted: what token 3 saw is what a chain of the three sees
    kept = [0, 1, 3]
    cache.write(kd[ctx:][kept], vd[ctx:][kept], slots[ctx:ctx + 3])  # quantising a value of the cache again: near it
    k2, _ = cache.read(slots[:ctx + 3], torch.float32)
    assert torch.equal(k2[:ctx], kd[:ctx])
    s = torch.einsum("hgd,nhd->hgn", q[3].view(heads, group, dim).double(), torch.cat([kd[:ctx], kd[ctx:][kept]]).double()) / 8.0
    dense = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), torch.cat([vd[:ctx], vd[ctx:][kept]]).double()).reshape(heads * group, dim)
    assert torch.allclose(y[3].double(), dense, rtol=0, atol=2.0 ** -16 * float(vd.abs().max()))


def test_refusals():
    kv = api()
    pages, table = filled(64, 2, 16, [20, 20], 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    q, k, s = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda"), torch.arange(2, device="cuda")
    bad = [
        (ValueError, lambda: kv.e8_cache_pages(1, 1, 16, 80)),
        (ValueError, lambda: kv.e8_cache_pages(1, 1, 24, 64)),
        (ValueError, lambda: kv.e8_cache_pages(1, 1, 8, 64)),
        (ValueError, lambda: kv.e8_cache_write(pages, k[:, :1], k[:, :1], s)),
        (ValueError, lambda: kv.e8_cache_write(pages, k, k[:1], s)),
        (ValueError, lambda: kv.e8_cache_write(pages, k, k, s[:1])),
        (ValueError, lambda: kv.e8_cache_write(pages, k.cpu(), k, s)),
        (ValueError, lambda: kv.e8_cache_write(pages, k, k, s.cpu())),
        (TypeError, lambda: kv.e8_cache_write(pages, k, k.bfloat16(), s)),
        (TypeError, lambda: kv.e8_cache_write(pages, k.half(), k.half(), s)),
        (TypeError, lambda: kv.e8_cache_write(pages, k, k, s.int())),
        (TypeError, lambda: kv.e8_cache_write(pages.float(), k, k, s)),
        (ValueError, lambda: kv.e8_cache_write(pages[..., :17], k, k, s)),
        (ValueError, lambda: kv.e8_cache_write(pages.transpose(0, 1), k, k, s)),
        (RuntimeError, lambda: kv.e8_cache_write(pages, k.clone().requires_grad_(), k, s)),
        (TypeError, lambda: kv.e8_cache_read(pages, s, torch.float16)),
        (TypeError, lambda: kv.e8_cache_read(pages, s.int())),
        (ValueError, lambda: kv.e8_cache_read(pages, s.view(1, 2))),
        (ValueError, lambda: kv.e8_cache_attention(q[:, :3], pages, t, n)),
        (ValueError, lambda: kv.e8_cache_attention(q[0], pages, t, n)),
        (ValueError, lambda: kv.e8_cache_attention(q[..., :32], pages, t, n)),
        (TypeError, lambda: kv.e8_cache_attention(q.half(), pages, t, n)),
        (ValueError, lambda: kv.e8_cache_attention(q[:1], pages, t, n)),
        (ValueError, lambda: kv.e8_cache_attention(q, pages, t[:1], n)),
        (TypeError, lambda: kv.e8_cache_attention(q, pages, t.long(), n)),
        (TypeError, lambda: kv.e8_cache_attention(q, pages, t, n.long())),
        (ValueError, lambda: kv.e8_cache_attention(q, pages, t, n, q_starts=n)),
        (ValueError, lambda: kv.e8_cache_attention(q, pages, t, n, tree=torch.zeros(1, dtype=torch.int64, device="cuda"))),
        (ValueError, lambda: kv.e8_cache_attention(torch.zeros(130, 4, 64, device="cuda"), pages, t, n, tree=torch.zeros(130, dtype=torch.int64, device="cuda"))),
        (ValueError, lambda: kv.e8_cache_attention(q, pages, t, n, out=q)),
        (ValueError, lambda: kv.e8_cache_attention(q, pages, t, n, out=q[:1])),
        (TypeError, lambda: kv.e8_cache_attention(q, pages, t, n, out=torch.zeros_like(q).bfloat16())),
        (RuntimeError, lambda: kv.e8_cache_attention(q.clone().requires_grad_(), pages, t, n)),
    ]
    before = pages.clone()
    for i, (kind, call) in enumerate(bad):
        with pytest.raises(kind):
            call()
            print("not refused:", i)
    assert torch.equal(before, pages)
    with torch.no_grad():
        kv.e8_cache_attention(q.clone().requires_grad_(), pages, t, n)
    with torch.inference_mode():
        made = kv.e8_cache_pages(2, 2, 16, 64)
        kv.e8_cache_write(made, k, k, s)
        kv.e8_cache_attention(q, made, t.clamp(max=1), n)
    kv.e8_cache_attention(q, pages, t, n)
