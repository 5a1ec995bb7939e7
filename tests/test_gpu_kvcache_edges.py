"""The E8-coded key/value cache at the edges of what its calls allow: layouts with dimensions of one, streams that are not PyTorch's own, long sums, values
of every size beside each other."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import kvcache_util as plain
from test_gpu_kvcache import DTYPES, api, as_words, check, expected_pages, filled, rows

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


def test_queries_that_are_none_are_refused():
    kv = api()
    pages, table = filled(64, 2, 16, [20, 20], 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    for kind, q in ((TypeError, None), (TypeError, [1.0]), (ValueError, torch.zeros((), device="cuda")), (ValueError, torch.zeros(2, 4, 0, device="cuda")),
                    (ValueError, torch.zeros(64, device="cuda"))):
        with pytest.raises(kind, match="q must"):
            kv.e8_cache_attention(q, pages, t, n)
    q = rows(2, 4, 64, 3).cuda()
    assert torch.equal(kv.e8_cache_attention(q, pages, t, n), kv.e8_cache_attention(q, pages, t, n, scale=0.125))


# ------------------------------------------------------------------ streams
def test_the_per_thread_default_stream_is_another_one_in_every_thread():
    """One handle, a stream for each thread: calls that run at the same time share nothing.  (The threads allocate nothing between their calls: PyTorch's
    allocator takes these streams for one.)"""
    import threading
    kv = api()
    dim, calls, tokens = 128, 60, (1, 9, 40)
    pages, table = filled(dim, 2, 16, [900, 300], 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([900, 300], dtype=torch.int32, device="cuda")
    qs = [[rows(2 * k, 8, dim, 10 * s + k, torch.bfloat16).cuda() for k in tokens] for s in range(4)]
    want = [[kv.e8_cache_attention(q, pages, t, n) for q in its] for its in qs]
    outs = [[[torch.zeros_like(q) for q in its] for _ in range(calls)] for its in qs]
    torch.cuda.synchronize()
    start, raised = threading.Barrier(4), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.ExternalStream(2)):  # cudaStreamPerThread
                start.wait(30)
                for out in outs[i]:
                    for q, y in zip(qs[i], out):
                        kv.e8_cache_attention(q, pages, t, n, out=y)
        except BaseException as e:
            raised.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    torch.cuda.synchronize()
    assert not raised
    for i in range(4):
        for out in outs[i]:
            assert all(torch.equal(y, w) for y, w in zip(out, want[i]))


def test_streams_that_come_and_go():
    """Streams made elsewhere, each used and destroyed: more of them than buffers are kept for, without one being held for each."""
    import ctypes
    kv = api()
    dim = 64
    pages, table = filled(dim, 2, 16, [700], 5)
    t, n = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([700], dtype=torch.int32, device="cuda")
    q = rows(1, 8, dim, 1, torch.bfloat16).cuda()
    want = kv.e8_cache_attention(q, pages, t, n)
    torch.cuda.synchronize()
    runtime, most = torch.cuda.cudart(), 0
    for i in range(400):
        handle = ctypes.c_void_p()
        assert int(runtime.cudaStreamCreate(ctypes.addressof(handle))) == 0
        with torch.cuda.stream(torch.cuda.ExternalStream(handle.value)):
            y = kv.e8_cache_attention(q, pages, t, n)
            torch.cuda.current_stream().synchronize()
        assert torch.equal(y, want)
        del y
        assert int(runtime.cudaStreamDestroy(handle.value)) == 0
        if i in (199, 399):
            most = torch.cuda.memory_allocated() - (most if i == 399 else 0)
    assert most <= 2 ** 20  # nothing is kept for the last 200


@pytest.mark.parametrize("dim, dtype, tokens", [(128, "bf16", 1), (64, "f32", 3), (128, "bf16", 40), (256, "bf16", 2)])
def test_the_first_call_of_a_process_may_be_captured(dim, dtype, tokens):
    import subprocess
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "kvcache_capture_child.py")
    done = subprocess.run([sys.executable, child, str(dim), dtype, str(tokens)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stdout + done.stderr


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_a_capture_that_forks_into_two_streams(tokens):
    """Two calls side by side in one graph, and one behind both."""
    kv = api()
    dim = 128
    pages, table = filled(dim, 2, 16, [900, 300], 5)
    t, lens = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([100, 60], dtype=torch.int32, device="cuda")
    qs = [rows(2 * tokens, 8, dim, s, torch.bfloat16).cuda() for s in range(3)]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        got = [kv.e8_cache_attention(qs[0], pages, t, lens)]
        with torch.cuda.stream(side):
            got.append(kv.e8_cache_attention(qs[1], pages, t, lens))
        main.wait_stream(side)
        got.append(kv.e8_cache_attention(qs[2], pages, t, lens))
    for now in ([900, 300], [64, 64], [577, 1]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        for _ in range(20):
            graph.replay()
        for q, y in zip(qs, got):
            assert torch.equal(y, kv.e8_cache_attention(q, pages, t, lens))


# ------------------------------------------------------------------ long sums
LONG = [("f32", 128, 1, 1), ("f32", 64, 2, 5), ("f32", 256, 1, 1), ("bf16", 128, 4, 1), ("bf16", 128, 4, 3), ("bf16", 256, 2, 1), ("bf16", 64, 8, 5), ("bf16", 64, 8, 32),
        ("bf16", 128, 8, 16), ("bf16", 128, 8, 32)]


@pytest.mark.parametrize("alike", [4096, 262144], ids=["keys in groups", "keys alike"])
@pytest.mark.parametrize("form", LONG, ids=lambda f: f"{f[0]}d{f[1]}g{f[2]}t{f[3]}")
def test_sums_over_long_sequences(form, alike):
    """More sequences than the chip has CTAs, so that one CTA sums 262144 tokens.  Where the values are the same for all tokens, or follow no key, the result is
    their mean whatever the weights are: scores' errors leave no trace, weights' roundings at most 2^-11 (bf16 queries: half a step of 11 bits) or 2^-22 of it, and the sums of
    weights and of results are to be float32 sums, which is 2^-18.  The mean of a bf16 result lies 2^-10 beside the border between two numbers: further than all of it."""
    dtype, dim, group, tokens = form
    kv = api()
    L, page, heads, seqs = 262144, 128, 2, 160
    pages = kv.e8_cache_pages(L // page, heads, page, dim)
    g = torch.Generator().manual_seed(7)
    k = rows((L + alike - 1) // alike, heads, dim, 1).repeat_interleave(alike, 0)[:L].clone()
    if alike > 4096:
        k[:256] *= 0.5  # the running maximum is another one than that of most
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").expand(seqs, -1)
    lens = torch.full((seqs,), L, dtype=torch.int32, device="cuda")
    q = rows(tokens, heads * group, dim, 2, DTYPES[dtype]).cuda()
    slots = torch.arange(L, device="cuda")
    border = 7.0 - 2.0 ** -6  # between two bf16 numbers, 2^-5 apart
    for mean in ((6.5,) if dtype == "f32" else (border * (1 - 2.0 ** -10), border * (1 + 2.0 ** -10))):
        sevens = round((mean - 6) * 4096)  # of 4096 tokens in a row
        place = torch.arange(L) % 4096
        v = torch.where((place + 1) * sevens // 4096 > place * sevens // 4096, 7.0, 6.0)[:, None, None].expand(L, heads, dim).clone()
        v[..., 0] = 7.0  # a step of 1
        if dtype == "f32":
            v[:] = 7.0 * (1 + torch.rand(1, heads, dim, generator=g))
        kv.e8_cache_write(pages, k.cuda(), v.cuda(), slots)
        y, z = kv.e8_cache_attention(q.repeat(seqs, 1, 1), pages, table, lens, return_lse=True, tree=torch.full((seqs * tokens,), -1, device="cuda"))
        y, z = y.view(seqs, tokens, heads, group, dim), z.view(seqs, tokens, heads, group)
        kd, vd = (x.double() for x in kv.e8_cache_read(pages, slots))
        if dtype == "f32":
            worst = float((y.double() / vd[0, :, None] - 1).abs().max())
            assert worst <= 2.0 ** -24 + 2 * 2.0 ** -22 + 2.0 ** -18, f"{worst} of the mean"
        else:
            assert abs(float(vd[:, 0, 1].mean()) - mean) < 2.0 ** -13 and (vd[..., 1:8] == vd[..., 1:2]).all()
            want = 7.0 if mean > border else 7.0 - 2.0 ** -5
            part = float((y[..., 1:8].float() != want).float().mean())
            assert part == 0.0, f"{part} of the results are on the wrong side"
        s = torch.einsum("thgd,nhd->thgn", q.double().view(tokens, heads, group, dim), kd) / math.sqrt(dim)
        reach = torch.einsum("thgd,nhd->thgn", q.double().abs().view(tokens, heads, group, dim), kd.abs()[::128]).amax(-1) / math.sqrt(dim)
        lse = torch.logsumexp(s, -1)
        bound = (2.0 ** -22 + (dim + 32) * 2.0 ** -24) * 4 * reach + 2.0 ** -20 + 2.0 ** -18 + 2.0 ** -22 * lse.abs()
        worst = float(((z.double() - lse) / bound).abs().max())
        assert worst <= 1.0, f"lse: {worst} of the bound"


# ------------------------------------------------------------------ sizes
FORMS = [("f32", 64, 2), ("f32", 256, 9), ("bf16", 128, 2), ("bf16", 128, 12), ("bf16", 256, 4), ("bf16", 128, 24), ("bf16", 64, 40), ("bf16", 128, 72)]
FORM = lambda f: f"{f[0]}d{f[1]}g{f[2]}"  # noqa: E731


def with_values(dim, L, v, page=16, seed=3):
    """One sequence of L tokens and one head: random keys, these values [L, dim]."""
    kv = api()
    pages, table = filled(dim, 1, page, [L], seed)
    slots = torch.tensor([table[0][i // page] * page + i % page for i in range(L)], device="cuda")
    kv.e8_cache_write(pages, rows(L, 1, dim, 30).cuda(), v.view(L, 1, dim).cuda(), slots)
    return pages, table


@pytest.mark.parametrize("size", [2.0 ** -99, 1e-30, 1e-28, 1e-26, 1e-20, 1e20, 1e30, 1e32])
@pytest.mark.parametrize("form", FORMS, ids=FORM)
def test_values_of_every_size(form, size):
    """All of a sequence's values of one size, from the smallest rows that are kept to the largest whose weights keep all their bits."""
    dtype, dim, group = form
    L = 300
    v = rows(L, 1, dim, 31)[:, 0]
    v = v / v.abs().amax(-1, keepdim=True) * (1.0 + torch.rand(L, 1, generator=torch.Generator().manual_seed(2))) * size * 2.0
    pages, table = with_values(dim, L, v)
    q = rows(2, group, dim, 32, DTYPES[dtype]).cuda()
    check(q, pages, dim, table, [L], [0, 2], None)


@pytest.mark.parametrize("size", [1e33, 1e35, 1e37, 1e38])
@pytest.mark.parametrize("form", FORMS, ids=FORM)
def test_values_near_the_end_of_the_type(form, size):
    """Above 7e31 small weights are lost and sums have fewer bits: of 300 weights as large as each other, as zero keys make them, at most 2^-17 each by then."""
    dtype, dim, group = form
    L = 300
    v = rows(L, 1, dim, 31)[:, 0].clamp(-3, 3) * size
    v[:, 0] = 3.0 * size
    pages, table = with_values(dim, L, v)
    kc, kh, vc, vh = plain.planes(as_words(pages), dim)
    q = torch.zeros(2, group, dim, dtype=DTYPES[dtype], device="cuda")
    y, z = api().e8_cache_attention(q, pages, torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([L], dtype=torch.int32, device="cuda"), return_lse=True)
    at = [(table[0][i // 16], i % 16) for i in range(L)]
    vd = torch.stack([plain.values(vc[p, 0, r], vh[p, 0, r]) for p, r in at])
    for i, n in ((0, L - 1), (1, L)):  # a chain of two
        want, spread = vd[:n].mean(0), vd[:n].abs().mean(0)
        bound = torch.finfo(DTYPES[dtype]).eps / 2 * want.abs() + (2.0 ** -18 + 2.0 ** -17) * spread
        assert ((y[i].cpu().double() - want).abs() <= bound).all()
        assert ((z[i].cpu().double() - math.log(n)).abs() <= 2.0 ** -17 + 2.0 ** -20).all()


@pytest.mark.parametrize("form", FORMS, ids=FORM)
def test_a_cache_of_zero_values_gives_zeros(form):
    dtype, dim, group = form
    L = 200
    pages, table = with_values(dim, L, torch.zeros(L, dim))
    q = (rows(2, group, dim, 32) * 6).to(DTYPES[dtype]).cuda()
    got = check(q, pages, dim, table, [L], [0, 2], None)
    assert not got[0].any()


@pytest.mark.parametrize("order", ["zeros first", "zeros last", "in turn"])
@pytest.mark.parametrize("small, large", [(0.0, 1e5), (0.0, 1e14), (0.0, 1e30), (1e-28, 1e12)])
@pytest.mark.parametrize("form", FORMS, ids=FORM)
def test_values_that_weigh_nothing_count_in_the_sum(form, small, large, order):
    """Runs of tokens whose values are zeros (as of tokens that only take up attention) or tiny, beside runs of large ones: the first run's share of the
    softmax's sum is as large as the second's."""
    dtype, dim, group = form
    L = 1024
    run = torch.arange(L) // 128 if order == "in turn" else torch.arange(L) // (L // 2)
    tiny = run % 2 == (1 if order == "zeros last" else 0)
    v = rows(L, 1, dim, 31)[:, 0].clamp(-3, 3) * torch.where(tiny, small, large)[:, None]
    pages, table = with_values(dim, L, v, page=64)
    q = rows(2, group, dim, 32, DTYPES[dtype]).cuda()
    check(q, pages, dim, table, [L], [0, 2], None)


@pytest.mark.parametrize("size", [1.0, 2.0 ** -99, 1e-29, 1e-28, 1e-26, 1e28, 1e30])
@pytest.mark.parametrize("form", FORMS, ids=FORM)
def test_many_small_weights_beside_a_large_one(form, size):
    """The first token weighs 2^10 to 2^26 times as much as each of the 131071 others, whose sum counts all the same, for values of every size.  All values are the
    same: results are that, but for weights' roundings (2^-11 for bf16 queries, 2^-22 else), float32 sums (2^-18), what each weight lacks below 2^-31 of the largest,
    and, in the run of tokens that the tensor cores sum up with the first one, 2^-23 of the sum per token: they line up products by the largest number and cut off
    what lies behind its 24 bits.  A run is 8 units of 32 tokens for float32 queries, 64 of them or 64 tiles of 128 tokens for bf16."""
    dtype, dim, group = form
    kv = api()
    L, page, heads, seqs = 131072, 128, 2, 160
    run = 256 if dtype == "f32" else 8192
    pages = kv.e8_cache_pages(L // page, heads, page, dim)
    k = torch.zeros(L, heads, dim)
    k[0, :, :2] = 7.0
    v = (rows(1, heads, dim, 4).clamp(-3, 3) * size).expand(L, heads, dim)
    kv.e8_cache_write(pages, k.cuda(), v.cuda(), torch.arange(L, device="cuda"))
    vd = kv.e8_cache_read(pages, torch.arange(1, device="cuda"))[1][0].cpu().double()
    more = torch.linspace(10, 26, heads * group).double()
    q = torch.zeros(heads * group, dim)
    q[:, :2] = (more * math.log(2) * math.sqrt(dim) / 14)[:, None]
    q = q.to(DTYPES[dtype]).cuda()
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").expand(seqs, -1)
    y, z = kv.e8_cache_attention(q.expand(seqs, -1, -1), pages, table, torch.full((seqs,), L, dtype=torch.int32, device="cuda"), return_lse=True)
    want = vd.repeat_interleave(group, 0)
    weight = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -22
    off = (y.cpu().double() - want).abs() / want.abs().clamp(min=1e-300)
    worst = float(torch.where(want == 0, y.cpu().double().abs(), off).max())
    assert worst <= torch.finfo(DTYPES[dtype]).eps / 2 + 2 * weight + 2.0 ** -18 + L * 2.0 ** -31 + run * 2.0 ** -23, f"{worst} of the value"
    s = q[:, 0].cpu().double() * 14 / math.sqrt(dim)
    lse = torch.logaddexp(s, torch.full_like(s, math.log(L - 1)))
    bound = (2.0 ** -22 + (dim + 32) * 2.0 ** -24) * 4 * s + 2.0 ** -20 + 2.0 ** -18 + 2.0 ** -22 * lse
    worst = float(((z.cpu().double() - lse).abs() / bound).max())
    assert worst <= 1.0, f"lse: {worst} of the bound"


# ------------------------------------------------------------------ the benchmark
def test_the_benchmark_sets_against_hbm_only_what_l2_cannot_hold():
    from coset_b200 import benchmarks
    l2 = torch.cuda.get_device_properties(0).L2_cache_size
    records = list(benchmarks.iter_kvcache())
    assert {r["bench"] for r in records} == {"kvcache_write", "kvcache_read", "kvcache_attention"}
    for r in records:
        assert r["ms"] > 0 and (r["inputs"] == "beyond L2") == (r["input_bytes"] >= 2 * l2) == ("frac_of_hbm" in r)
        assert r.get("frac_of_hbm", 0.5) < 1.1
