"""Plain implementation of the E8-coded key/value cache for the tests: whole numbers and 64 bits, one block after the other's definition, on the CPU."""
import math

import numpy as np
import torch

SMALLEST = 2.0 ** -100


def head_words(dim):
    return (dim + 127) // 128


def steps_of(x):
    """float32 [..., dim] -> (step float32 [..., 1], row kinds: 0 plain, 1 zeros, 2 no numbers)."""
    most = np.abs(x).max(-1, keepdims=True)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    small = ~bad & (most < SMALLEST)
    t = np.where(bad | small, np.float32(7), most).astype(np.float32) / np.float32(7)
    bits = t.view(np.uint32)
    step = ((bits.astype(np.uint64) + 0xFFFF) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return step, np.where(bad, 2, np.where(small, 1, 0))


def nearest(u):
    """int64 [n, 8] in units of 1/4096 -> (f, c): the nearest point of E8 is f + c / 2."""
    best = None
    for c in (0, 1):
        base = (u + 2048) // 4096 if c == 0 else u // 4096
        e = u - base * 4096 - 2048 * c
        wrong = base.sum(-1) % 2 != 0
        k = np.abs(e).argmax(-1)  # the first one
        move = np.where(np.take_along_axis(e, k[:, None], 1) > 0, 1, -1) * (np.arange(8) == k[:, None])
        f = base + np.where(wrong[:, None], move, 0)
        far = ((u - 4096 * f - 2048 * c) ** 2).sum(-1)
        if best is None:
            best = f, np.zeros(len(u), int), far
        else:
            nearer = far < best[2]
            best = np.where(nearer[:, None], f, best[0]), nearer.astype(int), np.where(nearer, far, best[2])
    return best[0], best[1]


def quantise(x):
    """Tensor [n, dim] (float32 or bf16, CPU) -> (codes uint32 [n, dim / 8], heads uint32 [n, words], values float64 [n, dim])."""
    x = x.float().numpy()
    n, dim = x.shape
    step, kind = steps_of(x)
    inv = np.float32(1) / step
    with np.errstate(all="ignore"):
        u = np.rint((x * inv).astype(np.float32).astype(np.float64) * 4096)
    u = np.where(kind == 0, u, 0).astype(np.int64)
    f, c = nearest(u.reshape(-1, 8))
    assert f.min() >= -8 and f.max() <= 7
    codes = ((f + 8).astype(np.uint64) << (4 * np.arange(8, dtype=np.uint64))).sum(-1).astype(np.uint32).reshape(n, dim // 8)
    c = c.reshape(n, dim // 8)
    bits = np.where(kind == 0, step.view(np.uint32), np.where(kind == 1, 0, 0x7FC00000)).astype(np.uint32)
    heads = np.empty((n, head_words(dim)), np.uint32)
    for w in range(head_words(dim)):
        part = c[:, 16 * w:16 * w + 16]
        heads[:, w] = bits[:, 0] | (part << np.arange(part.shape[1])).sum(-1).astype(np.uint32)
    s = np.where(kind == 0, step.astype(np.float64), np.where(kind == 1, 0.0, np.nan))
    return codes, heads, torch.from_numpy((f.reshape(n, dim) + 0.5 * np.repeat(c, 8, 1)) * s)


def planes(pages, dim):
    """uint32 array [P, H, S, W] -> views (key codes, key heads, value codes, value heads) [P, H, S, words]."""
    P, H, S, W = pages.shape
    flat, kb, hw = pages.reshape(P, H, S * W), dim // 8, head_words(dim)
    cut = lambda at, w: flat[:, :, at * S:(at + w) * S].reshape(P, H, S, w)  # noqa: E731
    return cut(0, kb), cut(2 * kb, hw), cut(kb, kb), cut(2 * kb + hw, hw)


def values(codes, heads):
    """What codes and heads stand for, float64."""
    n = (codes[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    block = np.arange(codes.shape[-1])
    c = (heads[..., block // 16] >> (block % 16).astype(np.uint32)) & 1
    step = (heads[..., :1] & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)
    with np.errstate(all="ignore"):
        return torch.from_numpy(((n.astype(np.float64) - 8 + 0.5 * c[..., None]).reshape(*codes.shape[:-1], 8 * codes.shape[-1])) * step)


def attend(q, pages, dim, table, lens, starts, tree, scale):
    """(out, lse, spread, reach) in float64: spread = sum P |v| plus what of weights too small to be held may be lacking, against which weights' errors
    count; reach = the largest sum of |q k| scale of a seen key, against which scores' errors count.

    Weights are held relative to the row's largest P_n max|v_n|, in floating point whose smallest number is 2^-31 of it: what a key adds may be lacking
    up to that, whatever the sum is.  check() multiplies spread by 2^-18 at least, so 2^-13 of the largest a key stands for 2^-31 of it here.  q [n, heads, dim] float64; pages uint32 [P, H, S, W]; table, lens, starts, tree: lists."""
    kc, kh, vc, vh = planes(pages, dim)
    P, H, S, _ = pages.shape
    n, heads, _ = q.shape
    out, lse = torch.full((n, heads, dim), math.nan, dtype=torch.float64), torch.full((n, heads), math.nan, dtype=torch.float64)
    spread, reach = torch.zeros(n, heads, dim, dtype=torch.float64), torch.zeros(n, heads, 1, dtype=torch.float64)
    for b in range(len(lens)):
        count = starts[b + 1] - starts[b]
        L = min(lens[b], len(table[b]) * S)
        at = [(table[b][i // S], i % S) for i in range(L)]
        there = torch.tensor([0 <= p < P for p, _ in at], dtype=torch.bool)
        p, r = np.array([max(0, min(x, P - 1)) for x, _ in at], int), np.array([y for _, y in at], int)
        for i in range(count):
            row = starts[b] + i
            j = torch.arange(L) - (L - count)
            if tree is None:
                seen = j <= i
            else:
                seen = (j < 0) | torch.tensor([0 <= x < 64 and bool(tree[row] >> int(x) & 1) for x in j], dtype=torch.bool)
            seen = seen & there
            for h in range(heads):
                g = h // (heads // H)
                k, v = values(kc[p, g, r], kh[p, g, r])[seen], values(vc[p, g, r], vh[p, g, r])[seen]
                if not len(k):
                    out[row, h], lse[row, h] = 0.0, -math.inf
                    continue
                s = (k @ q[row, h]) * scale
                lse[row, h] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[row, h])
                lost = len(k) * 2.0 ** -13 * (w * v.abs().amax(-1)).max()
                out[row, h], spread[row, h] = w @ v, w @ v.abs() + lost
                reach[row, h] = (k.abs() @ q[row, h].abs()).max() * abs(scale)
    return out, lse, spread, reach
