"""Operators of the E8-coded key/value cache: what a serving program has this package do with one.

  store   the keys and values of new tokens are quantised into the cache's pages (e8_cache_write) and read back as the values
          that the cache now stands for (e8_cache_read)
  read    cached tokens are read back as dense keys and values (e8_cache_read), as for a prompt that continues a cached prefix
  attend  softmax attention of one token, of a chain or of a tree of drafted tokens over the cache (e8_cache_attention)

A row is the D values of one token and one head (D = 64, 128 or 256).  Its step is the smallest bf16 number that is at least
max|x| / 7; its values in steps, rounded to 1/4096, are replaced by the nearest point of the lattice E8 block by block (8 values),
whose coordinates lie in [-8, 7.5]: f + c / 2 with f a 4-bit number per value and c a bit per block.

A page of one head is a record of words (int32): the codes of the S keys, D / 8 words each (value i of a block in bits 4i..4i+3, as
f + 8); the codes of the S values; the heads of the keys, one word per 128 values of a row: the step's 16 bits in the high half, the
blocks' bits c in the low half; the heads of the values.  The pages are [n_pages, n_heads, S, D / 4 + 2 ceil(D / 128)].

`own` false: elementary torch operations in 32 bits.  `own` true: the package's kernels.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one generation step of 32 sequences: the smallest call, made once per layer and step
        {"name": "store_step", "kind": "store", "n": 32, "heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a long prompt
        {"name": "store_prompt", "kind": "store", "n": 8192, "heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # twelve heads of 64 in float32, a length that is no multiple of anything, small pages, and tokens that are padding
        {"name": "store_f32_padded", "kind": "store", "n": 1003, "heads": 12, "dim": 64, "page": 16, "dtype": "f32", "padding": True},
        # a cached prefix handed to a dense attention
        {"name": "read_prefix", "kind": "read", "n": 32768, "heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # a few hundred tokens of wide heads in float32
        {"name": "read_f32_wide", "kind": "read", "n": 777, "heads": 4, "dim": 256, "page": 32, "dtype": "f32"},
        # generation: one short sequence (latency), a batch of long ones, one very long one
        {"name": "attend_one", "kind": "attend", "batch": 1, "tokens": 1, "lo": 1000, "hi": 1000, "heads": 8, "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "mask": "chain"},
        {"name": "attend_batch", "kind": "attend", "batch": 32, "tokens": 1, "lo": 4000, "hi": 8192, "heads": 8, "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "mask": "chain"},
        {"name": "attend_long", "kind": "attend", "batch": 1, "tokens": 1, "lo": 131071, "hi": 131071, "heads": 8, "group": 8, "dim": 128, "page": 128, "dtype": "bf16", "mask": "chain"},
        # twelve heads of 64 without grouping, float32
        {"name": "attend_f32", "kind": "attend", "batch": 3, "tokens": 1, "lo": 100, "hi": 512, "heads": 12, "group": 1, "dim": 64, "page": 16, "dtype": "f32", "mask": "chain"},
        # speculative decoding: small trees, large ones over long caches, and chains of different lengths with wide heads
        {"name": "tree_small", "kind": "attend", "batch": 8, "tokens": 8, "lo": 500, "hi": 3000, "heads": 8, "group": 4, "dim": 128, "page": 64, "dtype": "bf16", "mask": "tree"},
        {"name": "tree_large", "kind": "attend", "batch": 4, "tokens": 64, "lo": 8000, "hi": 16384, "heads": 8, "group": 8, "dim": 128, "page": 64, "dtype": "bf16", "mask": "tree"},
        {"name": "chains_ragged_wide", "kind": "attend", "batch": 5, "tokens": 13, "lo": 1, "hi": 2500, "heads": 4, "group": 2, "dim": 256, "page": 32, "dtype": "bf16", "mask": "chain", "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "attend", "attend", "attend"])
    case = {"kind": kind, "dim": rng.choice([64, 128, 128, 128, 256]), "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "f32"])}
    if kind != "attend":
        case["heads"] = rng.randint(1, 16)
        case["n"] = max(1, min(_log(rng, 1, 32768), (1 << 25) // (case["heads"] * case["dim"])))
        if kind == "store":
            case["n"] = min(case["n"], (1 << 23) // (case["heads"] * case["dim"]))
            case["padding"] = rng.random() < 0.3
        return case
    case["mask"] = rng.choice(["chain", "tree"])
    case["ragged"] = rng.random() < 0.3
    while True:
        case.update(batch=_log(rng, 1, 64), tokens=rng.choice([1, 1, rng.randint(2, 64)]), heads=rng.choice([1, 2, 4, 8, 8, 12, 16]), group=rng.choice([1, 2, 3, 4, 4, 6, 7, 8, 16]))
        case["hi"] = _log(rng, 16, 131072)
        case["lo"] = rng.choice([1, case["hi"], max(1, case["hi"] // 2), max(1, case["hi"] // 3)])
        w = work(case)
        if w["flops"] <= 1.3e11 and w["bytes"] <= 2.4e8 and case["batch"] * case["hi"] * case["heads"] * case["dim"] <= 1 << 28:
            return case


# ------------------------------------------------------------------ sizes that follow from a case alone
def _lengths(case):
    """(tokens in the cache, queried tokens among them) of each sequence."""
    lo, hi, T = case["lo"], case["hi"], case["tokens"]
    lens = [lo + int((hi - lo) * ((b + 1) * 0.6180339887 % 1.0)) for b in range(case["batch"])]
    lens[-1] = hi
    if not case.get("ragged"):
        return lens, [T] * case["batch"]
    return lens, [1 + (b * 7 + T - 1) % T for b in range(case["batch"])]


def _words(dim):
    """Words of a row's head."""
    return (dim + 127) // 128


# ------------------------------------------------------------------ the format, in elementary operations
def _quantise(x):
    """x [..., D] -> codes int32 [..., D / 8] and heads int32 [..., ceil(D / 128)]."""
    x = x.float()
    D = x.shape[-1]
    amax = x.abs().amax(-1, keepdim=True)
    t = amax / torch.full_like(amax, 7.0)  # by a tensor: an IEEE division
    step = ((t.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32)
    plain = (amax >= 2.0 ** -100) & torch.isfinite(amax)
    inv = torch.ones_like(step) / torch.where(plain, step, 1.0)
    u = torch.where(plain, torch.round(x * inv * 4096.0), 0.0).to(torch.int32).view(*x.shape[:-1], D // 8, 8)
    place = torch.arange(8, device=x.device, dtype=torch.int32)
    f = (u + 2048) >> 12
    d = u - (f << 12)
    a = d.abs()
    top, low = (a * 8 + 7 - place).amax(-1, keepdim=True), (a * 8 + place).amin(-1, keepdim=True)
    odd = (f.sum(-1, keepdim=True, dtype=torch.int32) & 1).bool()
    far = torch.where(odd, 4096 - 2 * (top >> 3), 0)
    whole = f + torch.where(odd & (7 - (top & 7) == place), torch.where(d > 0, 1, -1), 0)
    h = u >> 12
    odd = (h.sum(-1, keepdim=True, dtype=torch.int32) & 1).bool()
    half_far = 8192 - a.sum(-1, keepdim=True, dtype=torch.int32) + torch.where(odd, 2 * (low >> 3), 0)
    half = h + torch.where(odd & ((low & 7) == place), torch.where((d < 0) & (d > -2048), 1, -1), 0)
    c = half_far < far
    n = (torch.where(c, half, whole) + 8).to(torch.int64)
    codes = (n << (4 * place.to(torch.int64))).sum(-1)
    codes = torch.where(codes >= 1 << 31, codes - (1 << 32), codes).to(torch.int32)
    bits = torch.where(plain, step.view(torch.int32), torch.where(torch.isfinite(amax), 0, 0x7FC00000)).to(torch.int32)
    c = c.squeeze(-1).to(torch.int32)
    c = torch.nn.functional.pad(c, (0, -c.shape[-1] % 16)).view(*c.shape[:-1], _words(D), 16)
    cosets = (c << torch.arange(16, device=x.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
    return codes, bits | cosets


def _values(codes, heads):
    """What codes [..., D / 8] and heads [..., ceil(D / 128)] stand for, float32 [..., D]."""
    D = 8 * codes.shape[-1]
    n = (codes.unsqueeze(-1) >> (4 * torch.arange(8, device=codes.device, dtype=torch.int32))) & 15
    block = torch.arange(D // 8, device=codes.device)
    c = (heads[..., block // 16] >> (block % 16).to(torch.int32)) & 1
    step = (heads[..., :1] & ~0xFFFF).view(torch.float32)
    return ((n - 8).float() + 0.5 * c.unsqueeze(-1).float()).flatten(-2) * step


def _planes(pages, dim):
    """Views of the pages' four planes: codes and heads of the keys, codes and heads of the values, [n_pages, n_heads, S, words]."""
    P, H, S, _ = pages.shape
    flat, kb, hw = pages.view(P, H, -1), dim // 8, _words(dim)
    codes = [flat[..., i * S * kb:(i + 1) * S * kb].view(P, H, S, kb) for i in (0, 1)]
    heads = [flat[..., 2 * S * kb + i * S * hw:2 * S * kb + (i + 1) * S * hw].view(P, H, S, hw) for i in (0, 1)]
    return codes[0], heads[0], codes[1], heads[1]


# ------------------------------------------------------------------ inputs
def _rows(shape, g, channels):
    """Keys or values: normal, some channels several times as wide, some tokens larger than others."""
    x = torch.randn(shape, device="cuda", generator=g) * channels
    return x * torch.exp(0.3 * torch.randn(shape[:-1] + (1,), device="cuda", generator=g))


def _channels(heads, dim, g, spread):
    return torch.exp(spread * torch.randn(heads, 1, dim, device="cuda", generator=g))


def _filled(n_pages, heads, page, dim, g):
    """Pages whose every row holds a token."""
    pages = torch.empty(n_pages, heads, page, dim // 4 + 2 * _words(dim), dtype=torch.int32, device="cuda")
    kc, kh, vc, vh = _planes(pages, dim)
    wide = [_channels(heads, dim, g, 0.7), _channels(heads, dim, g, 0.2)]
    some = max(1, (1 << 24) // (heads * page * dim))
    for at in range(0, n_pages, some):
        n = min(some, n_pages - at)
        for codes, head, w in ((kc, kh, wide[0]), (vc, vh, wide[1])):
            codes[at:at + n], head[at:at + n] = _quantise(_rows((n, heads, page, dim), g, w))
    return pages


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, H, D, S, dtype = case["kind"], case["heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    s = {"kind": kind, "dim": D, "dtype": dtype}
    if kind != "attend":
        n = case["n"]
        n_pages = (n + S - 1) // S + 3
        # tokens of a sequence follow each other inside a page, the pages lie anywhere
        slots = (torch.randperm(n_pages, device="cuda", generator=g).unsqueeze(1) * S + torch.arange(S, device="cuda")).view(-1)[:n]
        if kind == "read":
            s.update(pages=_filled(n_pages, H, S, D, g), slots=slots)
            return s
        if case.get("padding"):
            slots = torch.where(torch.rand(n, device="cuda", generator=g) < 0.1, -1, slots)
        k, v = (_rows((H, n, D), g, _channels(H, D, g, w)).transpose(0, 1).to(dtype).contiguous() for w in (0.7, 0.2))
        s.update(pages=torch.zeros(n_pages, H, S, D // 4 + 2 * _words(D), dtype=torch.int32, device="cuda"), slots=slots, k=k, v=v)
        return s
    lens, counts = _lengths(case)
    most = max((n + S - 1) // S for n in lens)
    used = sum((n + S - 1) // S for n in lens)
    n_pages = used + 2
    order = torch.randperm(n_pages, device="cuda", generator=g)[:used].to(torch.int32)
    table, at = torch.zeros(len(lens), most, dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(lens):
        k = (n + S - 1) // S
        table[b, :k] = order[at:at + k]
        at += k
    N, T = sum(counts), max(counts)
    starts = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    tree = None
    if case["mask"] == "tree":  # every drafted token follows the root or one drafted before it
        pick = torch.rand(len(lens), T, device="cuda", generator=g).tolist()
        bits = []
        for b, n in enumerate(counts):
            seen = []
            for j in range(n):
                up = int(pick[b][j] * (j + 1)) - 1
                seen.append((seen[up] if up >= 0 else 0) | 1 << j)
            bits += [v - (1 << 64) if v >= 1 << 63 else v for v in seen]
        tree = torch.tensor(bits, dtype=torch.int64, device="cuda")
    q = torch.randn(N, H * case["group"], D, device="cuda", generator=g) * 1.5
    s.update(pages=_filled(n_pages, H, S, D, g), table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), q=q.to(dtype),
             starts=starts.cuda() if case.get("ragged") else None, tree=tree, most=T)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["kind"]
    if own:
        from coset_b200.kvcache import e8_cache_attention, e8_cache_read, e8_cache_write
        if kind == "attend":
            return e8_cache_attention(s["q"], s["pages"], s["table"], s["lens"], q_starts=s["starts"], tree=s["tree"], return_lse=True)
        if kind == "store":
            e8_cache_write(s["pages"], s["k"], s["v"], s["slots"])
        return e8_cache_read(s["pages"], s["slots"], s["dtype"])
    pages, D = s["pages"], s["dim"]
    planes = _planes(pages, D)
    if kind == "attend":
        return _attend(s, planes)
    S, slots = pages.shape[2], s["slots"]
    there = slots >= 0
    if kind == "store":
        page, row = slots[there] // S, slots[there] % S
        planes[0][page, :, row], planes[1][page, :, row] = _quantise(s["k"][there])
        planes[2][page, :, row], planes[3][page, :, row] = _quantise(s["v"][there])
    page, row = slots.clamp(min=0) // S, slots.clamp(min=0) % S
    there = there.view(-1, 1, 1)
    return tuple(torch.where(there, _values(c[page, :, row], h[page, :, row]), 0.0).to(s["dtype"]) for c, h in (planes[:2], planes[2:]))


def _attend(s, planes):
    q, table, lens, tree, T = s["q"], s["table"].long(), s["lens"].long(), s["tree"], s["most"]
    N, D = q.shape[0], q.shape[2]
    B, H, S = table.shape[0], planes[0].shape[1], planes[0].shape[2]
    L = table.shape[1] * S
    if s["starts"] is None:
        first, count = torch.arange(B, device="cuda") * T, torch.full((B,), T, device="cuda")
    else:
        first, count = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(T, device="cuda")
    real = i < count[:, None]                                        # [B, T]
    at = torch.where(real, first[:, None] + i, 0)
    rows = q.float()[at].view(B, T, H, -1, D).permute(0, 2, 1, 3, 4)  # [B, H, T, G, D]
    G = rows.shape[3]
    k, v = (_values(c[table], h[table]).permute(0, 2, 1, 3, 4).reshape(B, H, L, D) for c, h in (planes[:2], planes[2:]))
    key = torch.arange(L, device="cuda")
    drafted = key - (lens - count)[:, None]                          # [B, L]: which of the queried tokens a key belongs to
    if tree is None:
        seen = drafted[:, None] <= i[:, None]
    else:
        bit = (tree[at][:, :, None] >> drafted.clamp(0, 63)[:, None]) & 1
        seen = (drafted < 0)[:, None] | ((bit == 1) & (drafted < 64)[:, None])
    seen = seen & (key < lens[:, None])[:, None]                      # [B, T, L]
    score = (rows.reshape(B, H, T * G, D) @ k.transpose(2, 3)).view(B, H, T, G, L) / math.sqrt(D)
    score = score.masked_fill(~seen[:, None, :, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, H, T * G, L) @ v).view(B, H, T, G, D) / torch.where(total > 0, total, 1.0)
    lse = (most + torch.log(total)).squeeze(-1)
    put = at[real]
    y, z = torch.empty(N, H * G, D, device="cuda"), torch.empty(N, H * G, device="cuda")
    y[put] = out.permute(0, 2, 1, 3, 4).reshape(B, T, H * G, D)[real]
    z[put] = lse.permute(0, 2, 1, 3).reshape(B, T, H * G)[real]
    return y.to(s["dtype"]), z


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    D, H = case["dim"], case["heads"]
    wide, record = D * (4 if case["dtype"] == "f32" else 2), D // 2 + 4 * _words(D)
    if case["kind"] != "attend":  # dense keys and values in (store) and out, the record written or read, a slot per token
        dense = 2 * wide if case["kind"] == "store" else wide
        return {"bytes": case["n"] * (2 * H * (dense + record) + 8), "flops": 0}
    lens, counts = _lengths(case)
    rows = sum(counts) * H * case["group"]
    tables = 4 * (len(lens) + sum((n + case["page"] - 1) // case["page"] for n in lens)) + (8 * sum(counts) if case["mask"] == "tree" else 0)
    return {"bytes": 2 * H * record * sum(lens) + rows * (2 * wide + 4) + tables, "flops": 4 * H * case["group"] * D * sum(n * t for n, t in zip(lens, counts))}


# ------------------------------------------------------------------ the definition in 64 bits, written apart from the above
def _in_coset(y, z):
    """The nearest point to y of the coset of D8 that z's coordinates, each the nearest one by itself, belong to, and its squared distance."""
    e = y - z
    wrong = torch.remainder(z.sum(-1, keepdim=True), 2.0) != 0.0
    at = e.abs().sort(dim=-1, descending=True, stable=True).indices[..., :1]
    z = torch.where(wrong, z.scatter_add(-1, at, torch.where(e.gather(-1, at) > 0, 1.0, -1.0).to(z.dtype)), z)
    return z, (y - z).square().sum(-1, keepdim=True)


def _nearest(y):
    """The nearest point of E8 to y [..., 8] (float64, multiples of 1/4096): the nearer of the nearest points of D8 and of D8 + 1/2, that of D8 where both are equally far."""
    whole, far = _in_coset(y, torch.floor(y + 0.5))
    half, half_far = _in_coset(y, torch.floor(y) + 0.5)
    return torch.where(half_far < far, half, whole)


def _stored(x):
    """What x [..., D] stands for once it is in the cache, float64."""
    most = x.double().abs().amax(-1, keepdim=True)
    t = (most / 7.0).float()
    kept = t.bfloat16().float()
    step = torch.where(kept < t, torch.nextafter(kept.bfloat16(), torch.full_like(kept, math.inf).bfloat16()).float(), kept).double()
    inv = (1.0 / step).float().double()
    y = torch.round((x.double() * inv).float().double() * 4096.0) / 4096.0
    return _nearest(y.unflatten(-1, (-1, 8))).flatten(-2) * step


def _read(pages, dim, page, row):
    """Keys and values of the rows `row` of pages `page`, float64 [n, heads, dim]."""
    P, H, S, _ = pages.shape
    words, hw, kb = pages.view(P, H, -1)[page], _words(dim), dim // 8
    nibble, block = 16 ** torch.arange(8, device="cuda"), torch.arange(kb, device="cuda")

    def plane(first, width):
        at = first + row[:, None] * width + torch.arange(width, device="cuda")
        return words.gather(2, at[:, None].expand(-1, H, -1)).long() & 0xFFFFFFFF

    def dense(code, head):
        step = (head[..., :1] >> 16).to(torch.int16).view(torch.bfloat16).double()
        f = (torch.div(code[..., None], nibble, rounding_mode="floor") % 16).double() - 8.0
        c = (torch.div(head[..., block // 16], 2 ** (block % 16), rounding_mode="floor") % 2).double()
        return (f + 0.5 * c[..., None]).flatten(2) * step

    return dense(plane(0, kb), plane(2 * S * kb, hw)), dense(plane(S * kb, kb), plane(2 * S * kb + S * hw, hw))


def exact(case, seed):
    s = prepare(case, seed)
    D = case["dim"]
    if case["kind"] != "attend":
        slots, S = s["slots"], case["page"]
        if case["kind"] == "store":
            got = _stored(s["k"]), _stored(s["v"])
        else:
            got = _read(s["pages"], D, slots // S, slots % S)
        return tuple(torch.where(slots.view(-1, 1, 1) >= 0, x, 0.0) for x in got)
    lens, counts = _lengths(case)
    S, H, G = case["page"], case["heads"], case["group"]
    out, lse, at = [], [], 0
    for b, (n, T) in enumerate(zip(lens, counts)):
        place = torch.arange(n, device="cuda")
        k, v = _read(s["pages"], D, s["table"][b].long()[place // S], place % S)
        q = s["q"][at:at + T].double().view(T, H, G, D)
        score = torch.einsum("thgd,nhd->thgn", q, k) / D ** 0.5
        j = place - (n - T)  # which of the queried tokens a key belongs to
        if s["tree"] is None:
            seen = j <= torch.arange(T, device="cuda")[:, None]
        else:
            bits = torch.tensor([[0 <= i < T and word >> i & 1 for i in range(64)] for word in s["tree"][at:at + T].tolist()], dtype=torch.bool, device="cuda")
            seen = (j < 0) | bits[:, j.clamp(0, 63)]
        score = score.masked_fill(~seen[:, None, None], -math.inf)
        z = torch.logsumexp(score, -1)
        p = torch.exp(score - torch.where(z == -math.inf, 0.0, z)[..., None])
        out.append(torch.einsum("thgn,nhd->thgd", p, v).reshape(T, H * G, D))
        lse.append(z.reshape(T, H * G))
        at += T
    return torch.cat(out), torch.cat(lse)
