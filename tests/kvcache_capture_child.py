"""Run by test_gpu_kvcache_edges.py in a process of its own: the first call of the cache that the process makes is captured into a graph."""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from coset_b200 import kvcache as kv


def main(dim, dtype, tokens):
    heads, group, page, length = 2, 4, 16, 100
    torch.manual_seed(1)
    pages = kv.e8_cache_pages(8, heads, page, dim)
    k, v = (torch.randn(length, heads, dim, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(tokens, heads * group, dim, device="cuda").to(dtype)
    slots = torch.randperm(8 * page, device="cuda")[:length]
    table = torch.randperm(8, device="cuda").int()[None]
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")

    def step():
        kv.e8_cache_write(pages, k, v, slots)
        return (*kv.e8_cache_read(pages, slots, dtype), *kv.e8_cache_attention(q, pages, table, lens, return_lse=True))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    assert not pages.any(), "written before the graph ran"
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in got]
    assert all(torch.equal(x, y) for x, y in zip(got, step())), "a replay and an eager call differ"
    assert bool(got[2].any()) and bool(got[3].isfinite().all())


if __name__ == "__main__":
    main(int(sys.argv[1]), {"f32": torch.float32, "bf16": torch.bfloat16}[sys.argv[2]], int(sys.argv[3]))
    torch.cuda.synchronize()
    print("ok")
