"""The serving operators over the paged K/V cache, as cases to measure.

One verification step of drafted tokens runs them in this order: the pages and slots of the
new tokens (``plan``), the visibility bits of the drafted trees (``mask``), the new K/V rows
into the pools (``write``), attention of every drafted token over its request's cache
(``attn``), and the rows of the accepted path moved together (``accept``).

``run`` computes them with elementary torch operations, or, with ``own`` true, with the
calls a user makes of ``fa4_ring``.
"""

import math
import os
import sys

import torch

own = False

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": E4M3}


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one step of 256 running requests, a few drafted tokens each, over a kept block table
        {"name": "plan decode", "op": "plan", "batch": 256, "new": 8, "cached": 32768, "page": 64,
         "kept": True},
        # 64 prompts admitted at once, 128K tokens in small pages
        {"name": "plan prompts", "op": "plan", "batch": 64, "new": 4096, "cached": 0, "page": 16,
         "kept": False},
        # a handful of requests with a small tree each: latency
        {"name": "mask small", "op": "mask", "batch": 8, "nodes": 8},
        # a large batch with wide trees (several 64-bit words a row)
        {"name": "mask large", "op": "mask", "batch": 512, "nodes": 200},
        # the new rows of one decode step, cut out of a fused q|k|v projection: latency
        {"name": "write decode", "op": "write", "tokens": 64, "padded": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64},
        # the rows of a prompt batch, quantised on their way into an e4m3 cache
        {"name": "write prompts e4m3", "op": "write", "tokens": 65536, "padded": 37, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "e4m3", "page": 128},
        # a few requests with small trees: latency
        {"name": "accept small", "op": "accept", "batch": 4, "nodes": 8, "depth": 4,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64},
        # a large batch of wide trees over an e4m3 cache
        {"name": "accept large", "op": "accept", "batch": 256, "nodes": 64, "depth": 12,
         "kv_heads": 8, "dim": 128, "dtype": "e4m3", "page": 16},
        # two requests, short caches, small trees: latency
        {"name": "attn small tree", "op": "attn", "batch": 2, "nodes": 12, "cached_min": 700,
         "cached": 1500, "heads": 32, "kv_heads": 8, "dim": 64, "dtype": "f16", "page": 16},
        # plain decode: one token for each of 64 requests with caches of 1K to 32K tokens
        {"name": "attn decode", "op": "attn", "batch": 64, "nodes": 1, "cached_min": 1000,
         "cached": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64},
        # verification of wide trees over an e4m3 cache: the most arithmetic for a byte
        {"name": "attn trees e4m3", "op": "attn", "batch": 32, "nodes": 64, "cached_min": 1000,
         "cached": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "e4m3", "page": 128},
        # two very long requests: the cache of the repository's long-context configuration
        {"name": "attn long e4m3", "op": "attn", "batch": 2, "nodes": 8, "cached_min": 262144,
         "cached": 262144, "heads": 16, "kv_heads": 2, "dim": 256, "dtype": "e4m3", "page": 64},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "mask", "write", "accept", "attn", "attn", "attn"])
    page = rng.choice([16, 32, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 128, 256])
    dtype = rng.choice(["bf16", "f16", "e4m3"])
    if op == "plan":
        batch = _log(rng, 1, 1024)
        new = _log(rng, 1, max(1, min(8192, 131072 // batch)))
        cached = rng.choice([0, _log(rng, 1, max(1, min(65536, 2 ** 24 // batch)))])
        return {"op": op, "batch": batch, "new": new, "cached": cached, "page": page,
                "kept": rng.random() < 0.5}
    if op == "mask":
        nodes = _log(rng, 1, 256)
        return {"op": op, "batch": _log(rng, 1, min(512, 100000 // nodes)), "nodes": nodes}
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 67108864 // (kv_heads * dim)),
                "padded": rng.choice([0, 1, 29]), "heads": kv_heads * rng.choice([1, 2, 4]),
                "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page}
    if op == "accept":
        nodes = _log(rng, 1, 128)
        return {"op": op, "batch": _log(rng, 1, 256), "nodes": nodes,
                "depth": rng.randint(1, min(nodes, 16)), "kv_heads": rng.choice([1, 2, 4]),
                "dim": rng.choice([64, 128]), "dtype": dtype, "page": page}
    group = rng.choice([1, 2, 3, 4, 5, 8])
    case = {"op": op, "batch": _log(rng, 1, 96), "nodes": rng.choice([1, _log(rng, 2, 64)]),
            "cached_min": 0, "cached": _log(rng, 1, 262144), "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page}
    most = work(listed()[9])["bytes"] / 2, work(listed()[10])["flops"] / 2
    while case["cached"] > 1 and (work(case)["bytes"] > most[0] or work(case)["flops"] > most[1]):
        case["cached"] = case["cached"] * 2 // 3
    case["cached_min"] = rng.choice([0, case["cached"] // 3, case["cached"]])
    return case


def _spread(lo, hi, n):
    """n whole numbers evenly spread from lo to hi."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(c):
    """(tokens in the cache before the step, new tokens) of each request, before a seed
    shuffles the requests."""
    b = c["batch"]
    if c["op"] == "plan":
        return _spread(c["cached"] // 16, c["cached"], b), _spread(0 if c["kept"] else 1, c["new"], b)
    if c["op"] == "mask":
        return [0] * b, _spread((c["nodes"] + 1) // 2, c["nodes"], b)
    if c["op"] == "accept":
        return [(37 * i) % 500 for i in range(b)], _spread((c["nodes"] + 1) // 2, c["nodes"], b)
    return _spread(c["cached_min"], c["cached"], b), _spread((c["nodes"] + 1) // 2, c["nodes"], b)


def _words(c):
    return (c["nodes"] + 63) // 64


def _max_pages(c):
    cached, new = _lens(c)
    return (max(cached) + max(new) + c["page"] - 1) // c["page"]


def work(case):
    c, op = case, case["op"]
    if op == "write":
        el, row = (1 if c["dtype"] == "e4m3" else 2), c["kv_heads"] * c["dim"]
        n = c["tokens"]
        return {"bytes": 2 * n * row * (2 + el) + 8 * (n + c["padded"]), "flops": 2 * n * row}
    cached, new = _lens(c)
    total = sum(new)
    if op == "plan":
        touched = sum(-(-(a + b) // c["page"]) - a // c["page"] for a, b in zip(cached, new) if b)
        table = c["batch"] * _max_pages(c) * 4 * (2 if c["kept"] else 1)
        return {"bytes": table + 8 * total + 4 * touched + 24 * c["batch"], "flops": 0}
    if op == "mask":
        return {"bytes": total * (4 + 8 * _words(c)) + 4 * c["batch"], "flops": 0}
    if op == "accept":
        el, row = (1 if c["dtype"] == "e4m3" else 2), c["kv_heads"] * c["dim"]
        moved = sum(min(c["depth"], n) for n in new)
        return {"bytes": 2 * total * row * (2 + el) + 2 * moved * row * 2 * el + 12 * c["batch"],
                "flops": 0}
    el = 1 if c["dtype"] == "e4m3" else 2
    keys = sum(a + b for a, b in zip(cached, new))
    pairs = sum((a + 1) * b for a, b in zip(cached, new))
    rows = total * c["heads"]
    return {"bytes": keys * c["kv_heads"] * c["dim"] * 2 * el + rows * (c["dim"] * 4 + 4)
            + total * 8 * _words(c) + 4 * (keys // c["page"] + 3 * c["batch"]),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# --------------------------------------------------------------------------- inputs

def _cu(lens, dev):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)


def _values(shape, dtype, g, dev):
    """N(0, 1) rows of a cache or a query; an e4m3 cache holds x / descale, amax at 448."""
    if dtype == E4M3:
        x = torch.randn(shape, generator=g, device=dev, dtype=torch.bfloat16)
        return (x * 88).clamp_(-448, 448).to(E4M3)
    return torch.randn(shape, generator=g, device=dev, dtype=dtype)


def _tables(lens, c, rng, dev, spare=3):
    """Block table [batch, max_pages] of shuffled pages for `lens` tokens, and the pool's size."""
    counts = [-(-n // c["page"]) for n in lens]
    pages = sum(counts) + spare
    perm = torch.randperm(pages, generator=rng, dtype=torch.int32)
    table = torch.full((len(lens), max(_max_pages(c), 1)), -1, dtype=torch.int32)
    at = 0
    for j, n in enumerate(counts):
        table[j, :n] = perm[at:at + n]
        at += n
    return table.to(dev), pages, perm[at:].to(dev)


def prepare(case, seed):
    c, dev = dict(case), "cuda"
    rng = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"c": c}
    if c["op"] == "write":
        hq, hk, d, n = c["heads"], c["kv_heads"], c["dim"], c["tokens"] + c["padded"]
        src = torch.bfloat16 if c["dtype"] == "e4m3" else DTYPES[c["dtype"]]
        qkv = torch.randn(n, (hq + 2 * hk) * d, generator=g, device=dev, dtype=src)
        s["k"], s["v"] = (qkv[:, (hq + i * hk) * d:(hq + (i + 1) * hk) * d].view(n, hk, d) for i in (0, 1))
        pages = -(-c["tokens"] // c["page"]) + 3
        perm = torch.randperm(pages, generator=rng).to(dev)
        at = torch.arange(c["tokens"], device=dev)
        slots = perm[at // c["page"]] * c["page"] + at % c["page"]
        s["slots"] = torch.cat([slots, torch.full((c["padded"],), -1, device=dev)])
        s["pools"] = [_values((pages, c["page"], hk, d), DTYPES[c["dtype"]], g, dev) for _ in range(2)]
        s["descale"] = _descales(c, g, dev)
        return s
    cached, new = _lens(c)
    order = torch.randperm(c["batch"], generator=rng).tolist()
    # requests are shuffled whole, so that the work and the pools' size are the same for every seed
    cached, new = [cached[i] for i in order], [new[i] for i in order]
    s["tokens"] = sum(new)
    s["max_nodes"] = max(new)
    s["cached"] = torch.tensor(cached, dtype=torch.int32, device=dev)
    s["new"] = torch.tensor(new, dtype=torch.int32, device=dev)
    if c["op"] == "plan":
        table, pages, _ = _tables(cached, c, rng, dev, spare=0)
        s["max_pages"] = max(_max_pages(c), 1)
        s["table"] = table if c["kept"] else None
        need = sum(-(-(a + b) // c["page"]) for a, b in zip(cached, new)) + 11
        free = torch.randperm(need + pages, generator=rng, dtype=torch.int32)
        s["free"] = (free[free >= pages] if c["kept"] else free).to(dev)
        return s
    s["cu"] = _cu(new, dev)
    i = torch.cat([torch.arange(n) for n in new])
    s["parents"] = (torch.rand(i.shape, generator=rng) * (i + 1)).floor().to(torch.int32).to(dev) - 1
    if c["op"] == "mask":
        return s
    lens = [a + b for a, b in zip(cached, new)]
    s["table"], pages, _ = _tables(lens, c, rng, dev)
    hk, d = c["kv_heads"], c["dim"]
    s["pools"] = [_values((pages, c["page"], hk, d), DTYPES[c["dtype"]], g, dev) for _ in range(2)]
    s["descale"] = _descales(c, g, dev)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    src = torch.bfloat16 if c["dtype"] == "e4m3" else DTYPES[c["dtype"]]
    if c["op"] == "attn":
        s["max_len"] = max(lens)
        s["q"] = torch.randn(s["tokens"], c["heads"], d, generator=g, device=dev, dtype=src)
        s["mask"] = _plain_mask(s["parents"], s["cu"], s["max_nodes"]) if c["nodes"] > 1 else None
        return s
    s["k"], s["v"] = (torch.randn(s["tokens"], hk, d, generator=g, device=dev, dtype=src) for _ in range(2))
    at = torch.arange(s["tokens"], device=dev)
    req = torch.repeat_interleave(torch.arange(c["batch"], device=dev), s["new"])
    pos = s["cached"].long()[req] + at - s["cu"].long()[req]
    s["slots"] = s["table"].long()[req, pos // c["page"]] * c["page"] + pos % c["page"]
    # an increasing list of accepted nodes for each request, ended by -1
    depth = c["depth"]
    accepted = torch.full((c["batch"], depth), -1, dtype=torch.int32)
    for j, n in enumerate(new):
        m = min(depth, n)
        accepted[j, :m] = torch.randperm(n, generator=rng)[:m].sort().values
    s["accepted"] = accepted.to(dev)
    return s


def _descales(c, g, dev):
    if c["dtype"] != "e4m3":
        return None, None
    return tuple(0.009 + 0.004 * torch.rand(c["kv_heads"], generator=g, device=dev) for _ in range(2))


# --------------------------------------------------------------------------- plain forms

def _plain_plan(s):
    c, dev = s["c"], s["cached"].device
    ps, mp = c["page"], s["max_pages"]
    cached, new = s["cached"].long(), s["new"].long()
    old = s["table"] if s["table"] is not None else torch.full((c["batch"], mp), -1, dtype=torch.int32, device=dev)
    col = torch.arange(mp, device=dev)
    used = (col >= (cached // ps)[:, None]) & (col < ((cached + new + ps - 1) // ps)[:, None]) & (new > 0)[:, None]
    want = used & (old < 0)
    rank = torch.cumsum(want.flatten(), 0).view_as(want) - 1
    have = s["free"].numel()
    got = want & (rank < have)
    table = torch.where(got, s["free"][rank.clamp(0, have - 1)], old)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    cu = torch.cat([zero, torch.cumsum(new, 0)])
    lens = cached + new
    cu_k = torch.cat([zero, torch.cumsum(lens, 0)])
    t = torch.arange(s["tokens"], device=dev)
    req = torch.searchsorted(cu[1:], t, right=True)
    pos = cached[req] + t - cu[req]
    page = table[req, pos // ps].long()
    slots = torch.where(page < 0, -1, page * ps + pos % ps)
    taken = torch.stack([got.sum(), want.sum() - got.sum()])
    i32 = torch.int32
    return table, slots, cu.to(i32), cu_k.to(i32), lens.to(i32), taken.to(i32)


def _plain_mask(parents, cu, max_nodes):
    """Ancestor closure by squaring the one-step relation, packed into 64-bit words."""
    dev, b, n = parents.device, cu.numel() - 1, max_nodes
    i = torch.arange(n, device=dev)
    lens = (cu[1:] - cu[:-1]).long()
    inside = i < lens[:, None]
    at = (cu[:-1].long()[:, None] + i).clamp(max=parents.numel() - 1)
    par = torch.where(inside, parents[at].long(), -1)
    reach = ((par[:, :, None] == i) | (i[:, None] == i)).to(torch.float32)
    for _ in range(max(1, (n - 1).bit_length())):
        reach = (torch.bmm(reach, reach) > 0).to(torch.float32)
    words = (n + 63) // 64
    bits = torch.zeros(b, n, words * 64, dtype=torch.int64, device=dev)
    bits[:, :, :n] = reach.to(torch.int64)
    packed = (bits.view(b, n, words, 64) << torch.arange(64, device=dev)).sum(-1)
    return packed[inside]


def _stored(x, descale, dtype):
    if dtype != E4M3:
        return x.to(dtype)
    return (x.float() / descale[:, None]).clamp(-448, 448).to(E4M3)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


def _plain_write(s):
    ok = s["slots"] >= 0
    for pool, x, descale in zip(s["pools"], (s["k"], s["v"]), s["descale"]):
        flat = _bytes(pool).view((-1,) + tuple(pool.shape[2:]))
        flat[s["slots"][ok]] = _bytes(_stored(x[ok], descale, pool.dtype))


def _plain_accept(s):
    c, acc = s["c"], s["accepted"].long()
    good = torch.cumprod(((acc >= 0) & (acc < s["new"].long()[:, None])).long(), 1).bool()
    cached = s["cached"].long()[:, None]

    def slot(pos):
        return s["table"].long().gather(1, pos // c["page"]) * c["page"] + pos % c["page"]

    src = slot(torch.where(good, cached + acc, 0))[good]
    dst = slot(torch.where(good, cached + torch.arange(acc.shape[1], device=acc.device), 0))[good]
    for pool in s["pools"]:
        flat = _bytes(pool).view((-1,) + tuple(pool.shape[2:]))
        flat[dst] = flat[src]
    return (s["cached"] + good.sum(1)).to(torch.int32)


def _plain_attn(s):
    c = s["c"]
    h, hk, d, n, size = c["heads"], c["kv_heads"], c["dim"], s["max_nodes"], s["max_len"]
    g, b, dev = h // hk, c["batch"], s["q"].device
    cu, lens, cached = s["cu"].long(), s["lens"].long(), s["cached"].long()
    i = torch.arange(n, device=dev)
    inside = i < s["new"][:, None]
    at = (cu[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][at].float().view(b, n, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * n, d)
    pages = s["table"].clamp(min=0).long()
    k, v = (_bytes(p)[pages].view(p.dtype).view(b, -1, hk, d)[:, :size].float() for p in s["pools"])
    if s["descale"][0] is not None:
        k, v = (x * e[:, None] for x, e in zip((k, v), s["descale"]))
    pos = torch.arange(size, device=dev)
    v = torch.where((pos < lens[:, None])[:, :, None, None], v, 0.0)
    node = pos - cached[:, None]
    seen = (node < 0)[:, None].expand(b, n, size)
    if s["mask"] is None:
        seen = seen | (node[:, None] <= i[:, None])
    else:
        word = s["mask"][at].gather(2, (node.clamp(min=0) // 64).clamp(max=s["mask"].shape[1] - 1)[:, None].expand(b, n, size))
        seen = seen | ((word >> (node.clamp(min=0) % 64)[:, None]) & 1).bool()
    seen = seen & (pos < lens[:, None])[:, None]
    score = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    score = score.view(b, hk, g, n, size).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hk, g * n, size), v.permute(0, 2, 1, 3)).view(b, hk, g, n, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)
    lse = (top + torch.log(total)).permute(0, 3, 1, 2, 4).reshape(b, n, h)
    return out[inside].to(s["q"].dtype), lse[inside]


# --------------------------------------------------------------------------- one pass

def _library():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fa4-cp_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import fa4_ring
    return fa4_ring


def run(state):
    s, op = state, state["c"]["op"]
    if not own:
        if op == "plan":
            return _plain_plan(s)
        if op == "mask":
            return _plain_mask(s["parents"], s["cu"], s["max_nodes"])
        if op == "attn":
            return _plain_attn(s)
        _plain_write(s)
        return s["pools"] + ([_plain_accept(s)] if op == "accept" else [])
    fa4 = _library()
    if op == "plan":
        p = fa4.paged_block_tables(s["cached"], s["new"], s["free"], page_size=s["c"]["page"],
                                   num_tokens=s["tokens"], block_table=s["table"],
                                   max_pages=s["max_pages"])
        return p.block_table, p.slot_mapping, p.cu_seqlens_q, p.cu_seqlens_k, p.seq_lens, p.pages
    if op == "mask":
        return fa4.paged_tree_mask(s["parents"], s["cu"], max_nodes=s["max_nodes"])
    k_pages, v_pages = s["pools"]
    kd, vd = s["descale"]
    if op == "attn":
        return fa4.b200_attn_paged_tree(
            s["q"], k_pages, v_pages, s["table"], cu_seqlens_q=s["cu"], seq_lens=s["lens"],
            max_seqlen_q=s["max_nodes"], tree_mask=s["mask"], k_descale=kd, v_descale=vd)
    fa4.paged_kv_write(s["k"], s["v"], k_pages, v_pages, s["slots"], k_descale=kd, v_descale=vd)
    if op == "write":
        return [k_pages, v_pages]
    lens = fa4.paged_kv_accept(k_pages, v_pages, s["table"], s["cached"], s["accepted"],
                               cu_seqlens_q=s["cu"])
    return [k_pages, v_pages, lens]


# --------------------------------------------------------------------------- 64 bits

def _exact_pools(s):
    """The pools after the write, request by request and in float64 (e4m3: the nearest e4m3
    value of the 64-bit quotient)."""
    done = []
    for pool, x, descale in zip(s["pools"], (s["k"], s["v"]), s["descale"]):
        rows = x.double()
        if pool.dtype == E4M3:
            rows = (rows / descale.double()[None, :, None]).clamp(-448, 448).to(E4M3)
        flat = pool.double().reshape((-1,) + tuple(pool.shape[2:]))
        keep = torch.nonzero(s["slots"] >= 0).flatten()
        flat.index_copy_(0, s["slots"][keep], rows.double()[keep])
        done.append(flat)
    return done


def _exact_attn(s):
    c = s["c"]
    h, hk, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    out = torch.zeros(s["tokens"], h, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["tokens"], h, dtype=torch.float64, device="cuda")
    cu, lens, cached = s["cu"].tolist(), s["lens"].tolist(), s["cached"].tolist()
    parents = s["parents"].tolist()
    for j in range(c["batch"]):
        a, n, size = cu[j], cu[j + 1] - cu[j], lens[j]
        pos = torch.arange(size, device="cuda")
        row = s["table"][j].long()[pos // ps] * ps + pos % ps
        k, v = (_bytes(p).reshape(-1, hk, d)[row].view(p.dtype).double() for p in s["pools"])
        if s["descale"][0] is not None:
            k, v = k * s["descale"][0].double()[:, None], v * s["descale"][1].double()[:, None]
        seen = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            if s["mask"] is None:
                seen[i, :i + 1] = True
                continue
            up = parents[a + i]
            if up >= 0:
                seen[i] = seen[up]
            seen[i, i] = True
        block = torch.zeros(n, size, dtype=torch.bool, device="cuda")
        block[:, :cached[j]] = True
        block[:, cached[j]:] = seen.to("cuda")
        for head in range(h):
            x = s["q"][a:a + n, head].double() @ k[:, head // (h // hk)].T / math.sqrt(d)
            x = x.masked_fill(~block, -math.inf)
            l = torch.logsumexp(x, 1)
            lse[a:a + n, head] = l
            out[a:a + n, head] = torch.exp(x - l[:, None]) @ v[:, head // (h // hk)]
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("plan", "mask"):
        return None
    if op == "attn":
        return _exact_attn(s)
    pools = _exact_pools(s)
    if op == "accept":
        ps, table = case["page"], s["table"].tolist()
        cached, new = s["cached"].tolist(), s["new"].tolist()
        src, dst = [], []
        for j, nodes in enumerate(s["accepted"].tolist()):
            for i, node in enumerate(nodes):
                if not 0 <= node < new[j]:
                    break
                for at, to in ((cached[j] + node, src), (cached[j] + i, dst)):
                    to.append(table[j][at // ps] * ps + at % ps)
        src, dst = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in (src, dst))
        pools = [p.index_copy(0, dst, p[src]) for p in pools]
    pools = [p.view(q.shape) for p, q in zip(pools, s["pools"])]
    return pools + ([None] if op == "accept" else [])
