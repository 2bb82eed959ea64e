"""Block tables and slot maps, tree masks, cache writes and accepted paths
(``fa4_ring.paged_cache``) against plain loops, and a serving loop of all of them."""

import math

import pytest
import torch

import paged_helpers as ph
from gpu_helpers import assert_device_ok

pytestmark = pytest.mark.gpu

BF, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def plain_plan(cached, new, free, page, num_tokens, table, width):
    """The definition, request by request."""
    table = [[-1] * width for _ in cached] if table is None else [list(r) for r in table]
    used = missing = 0
    slots = [-1] * num_tokens
    t = 0
    for j, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        for e in range(c // page, -(-(c + n) // page) if n else 0):
            if e < width and table[j][e] >= 0:
                continue
            if e < width and used < len(free):
                table[j][e] = free[used]
                used += 1
            else:
                missing += 1
        for i in range(n):
            e, r = divmod(c + i, page)
            if t < num_tokens and e < width and table[j][e] >= 0:
                slots[t] = table[j][e] * page + r
            t += 1
    lens = [max(c, 0) + max(n, 0) for c, n in zip(cached, new)]
    return table, slots, ph.cu_of([max(n, 0) for n in new]).tolist(), ph.cu_of(lens).tolist(), lens, [used, missing]


def check_plan(cached, new, free, page, width, table=None, num_tokens=None, num_free=None):
    from fa4_ring import paged_block_tables
    total = sum(max(n, 0) for n in new) if num_tokens is None else num_tokens
    p = paged_block_tables(i32(cached), i32(new), i32(free), page_size=page, num_tokens=total,
                           block_table=None if table is None else i32(table), max_pages=width,
                           num_free=None if num_free is None else i32([num_free]))
    want = plain_plan(cached, new, free if num_free is None else free[:num_free], page, total, table, width)
    for name, got, exp in zip(p._fields, p, want):
        assert got.cpu().tolist() == exp, name
    assert_device_ok()


def test_plan_small_cases():
    check_plan([0], [1], [7], 16, 1)
    check_plan([0], [0], [], 16, 3)
    check_plan([15, 16, 0, 17], [1, 1, 40, 0], [9, 8, 7, 6, 5, 4, 3], 16, 4)
    check_plan([15, 16, 3], [2, 31, 0], [9, 8, 7], 16, 4, [[1, -1, -1, -1], [2, -1, -1, -1], [3, -1, -1, -1]])
    check_plan([15, 16, 3], [2, 31, 9], [9, 8, 7], 16, 4, [[1, 4, -1, -1], [2, 5, 6, -1], [3, 0, -1, -1]])
    check_plan([-5, 2], [3, -7], [1, 2], 1, 4)                        # page size 1, negative lengths
    check_plan([5, 2], [3, 4], [1, 2, 3], 4, 3, num_tokens=12)         # padding behind the requests
    check_plan([5, 2], [3, 4], [1, 2, 3], 4, 3, num_tokens=5)          # more tokens than slots
    check_plan([0, 0, 0], [33, 33, 33], [1, 2, 3, 4], 16, 4)           # too few free pages
    check_plan([0, 60], [70, 9], list(range(20)), 16, 4)               # rows too narrow
    check_plan([200], [9], list(range(20)), 16, 4)                     # a cache past its row
    check_plan([0, 0], [40, 40], list(range(9)), 16, 4, num_free=2)
    check_plan([0, 0], [40, 40], list(range(9)), 16, 4, num_free=0)


@pytest.mark.parametrize("batch,page,top,grow", [(3, 64, 5000, 300), (200, 16, 900, 9), (1024, 16, 300, 40),
                                                 (1025, 32, 100, 3), (2500, 16, 64, 2), (2, 16, 10, 70000),
                                                 (40, 24, 3000, 2000)])
@pytest.mark.parametrize("kept", [False, True])
def test_plan_random(batch, page, top, grow, kept):
    g = torch.Generator().manual_seed(batch + page + kept)
    cached = torch.randint(0, top, (batch,), generator=g).tolist() if kept else [0] * batch
    new = torch.randint(0, grow + 1, (batch,), generator=g).tolist()
    width = -(-(max(cached) + max(new)) // page) + 1
    table = None
    if kept:  # pages of the cache, and of some requests a few more (left by rejected drafts)
        extra = torch.randint(0, 80, (batch,), generator=g).tolist()
        have = [min(-(-c // page) + (x if x < 40 else 0), width) for c, x in zip(cached, extra)]
        table = ph.block_table([h * page for h in have], page, g, width=width)[0].tolist()
    free = (torch.randperm(sum(-(-n // page) + 1 for n in new), generator=g) + 10 ** 6).tolist()
    check_plan(cached, new, free, page, width, table)


def test_plan_leaves_its_inputs_and_replays_in_a_graph():
    from fa4_ring import paged_block_tables
    cached, new, free = i32([3, 30]), i32([4, 4]), i32([5, 6, 7])
    table = i32([[0, -1, -1], [1, 2, -1]])
    before = [t.clone() for t in (cached, new, free, table)]

    def step():
        return paged_block_tables(cached, new, free, page_size=16, num_tokens=10, block_table=table)
    step()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        p = step()
    for c, n in (([3, 30], [4, 4]), ([16, 31], [1, 2]), ([0, 32], [0, 10])):
        cached.copy_(i32(c)); new.copy_(i32(n))
        gr.replay()
        want = plain_plan(c, n, [5, 6, 7], 16, 10, before[3].cpu().tolist(), 3)
        for got, exp in zip(p, want):
            assert got.cpu().tolist() == exp
    assert torch.equal(free, before[2]) and torch.equal(table, before[3])


@pytest.mark.parametrize("new,max_nodes", [([1], 1), ([8] * 5, 8), ([0, 64, 3, 65, 1], 65), ([200, 7, 129], 256),
                                           ([1000, 2], 1000), ([63] * 300, 63)])
def test_tree_mask(new, max_nodes):
    from fa4_ring import paged_tree_mask
    g = torch.Generator().manual_seed(sum(new))
    parents, cu = ph.random_parents(new, g), ph.cu_of(new)
    words = (max_nodes + 63) // 64
    want = torch.cat([ph.pack(ph.seen_of(parents, cu, j), words) for j in range(len(new))])
    pad = torch.full((3,), 5, dtype=torch.int32)
    got = paged_tree_mask(torch.cat([parents, pad]).cuda(), cu.cuda(), max_nodes=max_nodes)
    assert torch.equal(got[:-3].cpu(), want) and not got[-3:].any()
    chain = torch.cat([torch.arange(n, dtype=torch.int32) - 1 for n in new])
    got = paged_tree_mask(chain.cuda(), cu.cuda(), max_nodes=max_nodes)
    want = torch.cat([ph.pack(torch.tril(torch.ones(n, n)).bool(), words) for n in new])
    assert torch.equal(got.cpu(), want)
    assert_device_ok()


def test_tree_mask_bad_parents_and_sizes():
    from fa4_ring import paged_tree_mask
    # a later parent, itself, a huge and a very negative one: none of them
    got = paged_tree_mask(i32([1, 1, 10 ** 9, -2 ** 31, 0]), i32([0, 5]), max_nodes=5)
    assert got.cpu().flatten().tolist() == [1, 2, 4, 8, 17]
    # nodes past max_nodes see nothing; rows before the first and behind the last tree are 0
    got = paged_tree_mask(i32([-1] + [-1] * 70), i32([1, 70]), max_nodes=64)
    assert got.cpu().flatten().tolist()[:3] == [0, 1, 2]
    assert not got[65:].any()
    with pytest.raises(ValueError):
        paged_tree_mask(i32([0]), i32([0, 1]), max_nodes=0)
    with pytest.raises(ValueError):
        paged_tree_mask(i32([0]), i32([0, 1]), max_nodes=4097)
    assert paged_tree_mask(i32([]), i32([0, 0]), max_nodes=4).shape == (0, 1)


def stored(x, d, dt):
    """The definition in 64 bits: the nearest e4m3 value of the quotient, saturated."""
    if dt != E4M3 or x.dtype == E4M3:
        return x.to(dt)
    return (x.double() / d.double()[:, None]).clamp(-448, 448).to(E4M3)


@pytest.mark.parametrize("src,dst", [(BF, BF), (F16, F16), (BF, E4M3), (F16, E4M3), (E4M3, E4M3)])
@pytest.mark.parametrize("T,hk,D,page", [(1, 1, 64, 16), (77, 3, 128, 32), (300, 8, 256, 128), (5, 2, 48, 1)])
def test_write(src, dst, T, hk, D, page):
    from fa4_ring import paged_kv_write
    g = torch.Generator().manual_seed(T + D)
    pages = -(-T // page) + 3
    rows = (torch.randn(T, 5 * hk * D, generator=g) * 9).to(src)  # a fused projection
    k, v = rows[:, hk * D:2 * hk * D].view(T, hk, D), rows[:, 3 * hk * D:4 * hk * D].view(T, hk, D)
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[::7] = -1
    if T > 3:
        slots[1], slots[2] = pages * page, 2 ** 40  # outside the pools: skipped
    kd, vd = (0.01 + 0.05 * torch.rand(hk, generator=g) for _ in range(2))
    quant = dst == E4M3 and src != E4M3
    want, got = [], []
    for x, d in ((k, kd), (v, vd)):
        pool = (torch.randn(pages, page, hk, D, generator=g)).to(dst)
        got.append(pool.cuda())
        flat = pool.clone().view(torch.uint8).view(pages * page, hk, -1)
        ok = (slots >= 0) & (slots < pages * page)
        flat[slots[ok]] = stored(x, d, dst)[ok].contiguous().view(torch.uint8)
        want.append(flat.view(torch.uint8).view(pages, page, hk, -1))
    fused = rows.cuda()
    paged_kv_write(fused[:, hk * D:2 * hk * D].view(T, hk, D), fused[:, 3 * hk * D:4 * hk * D].view(T, hk, D),
                   got[0], got[1], slots.cuda(), k_descale=kd.cuda() if quant else None,
                   v_descale=vd.cuda() if quant else None)
    for a, b in zip(got, want):
        a = a.view(torch.uint8).cpu()
        if quant:  # -0 and the rare double rounding of the 64-bit quotient aside, the same bytes
            assert torch.equal(a.view(E4M3).double(), b.view(E4M3).double())
        else:
            assert torch.equal(a, b)
    assert_device_ok()


def test_write_saturates_and_keeps_nan():
    from fa4_ring import paged_kv_write
    x = torch.tensor([1e30, -1e30, math.inf, -math.inf, math.nan, 448, 465, 2 ** -10] * 8, dtype=BF).view(1, 1, 64)
    pool = torch.zeros(1, 1, 1, 64, dtype=E4M3, device="cuda")
    paged_kv_write(x.cuda(), x.cuda(), pool, pool.clone(), torch.zeros(1, dtype=torch.int64).cuda())
    got = pool.float().flatten()[:8].cpu()
    assert got[:4].tolist() == [448, -448, 448, -448] and math.isnan(got[4])
    assert got[5:].tolist() == [448, 448, 0.0]  # 2^-10: half of the smallest subnormal, to even


def test_write_layouts_offsets_and_empty():
    from fa4_ring import paged_kv_write
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(6, 2, 128, generator=g).to(BF).cuda() for _ in range(2))
    slots = torch.tensor([3, 17, 31, 0, 40, 8]).cuda()
    ref = torch.zeros(2, 3, 16, 2, 128, dtype=BF, device="cuda")
    paged_kv_write(k, v, ref[0], ref[1], slots)
    for make in (lambda: torch.zeros(3, 2, 16, 2, 128, dtype=BF, device="cuda").unbind(1),
                 lambda: [t.transpose(1, 2) for t in torch.zeros(2, 3, 2, 16, 128, dtype=BF, device="cuda")]):
        kp, vp = make()
        paged_kv_write(k, v, kp, vp, slots)
        assert torch.equal(kp, ref[0]) and torch.equal(vp, ref[1])
    odd = torch.randn(6, 1 + 2 * 128).to(BF).cuda()  # unaligned rows are copied first
    odd[:, 1:] = k.view(6, -1)
    kp, vp = torch.zeros_like(ref[0]), torch.zeros_like(ref[1])
    paged_kv_write(odd[:, 1:].view(6, 2, 128), v, kp, vp, slots)
    assert torch.equal(kp, ref[0])
    paged_kv_write(k[:0], v[:0], kp, vp, slots[:0])
    # a slot whose rows start past 2^32 elements
    pages = 2 ** 32 // (16 * 2 * 128) + 2
    big = torch.zeros(2, pages, 16, 2, 128, dtype=BF, device="cuda")
    paged_kv_write(k, v, big[0], big[1], slots + (pages - 3) * 16)
    assert torch.equal(big[:, -3:], ref)
    assert_device_ok()


@pytest.mark.parametrize("dt,D,page,hk", [(BF, 128, 16, 2), (F16, 64, 64, 1), (E4M3, 128, 32, 8), (E4M3, 16, 1, 1)])
def test_accept(dt, D, page, hk):
    from fa4_ring import paged_kv_accept
    g = torch.Generator().manual_seed(D + page)
    new = [1, 8, 64, 0, 30, 5, 40, 6]
    cached = [0, 15, 100, 20, 3, 16, 1, 7]
    lens = [a + b for a, b in zip(cached, new)]
    table, pages = ph.block_table(lens, page, g)
    acc = torch.full((8, 40), -1)
    lists = [[0], [1, 2, 7], [0, 5, 9, 10, 11, 12, 13, 20, 30, 63], [0], list(range(30)), [],
             list(range(1, 40)), [2, 1, 3]]
    counts = [1, 3, 10, 0, 30, 0, 39, 1]  # a list ends where it descends or leaves the tree
    for j, l in enumerate(lists):
        acc[j, :len(l)] = torch.tensor(l, dtype=torch.int64)
    pools, want = [], []
    for _ in range(2):
        pool = (torch.randn(pages, page, hk, D, generator=g) * 8).to(dt)
        pools.append(pool.cuda())
        flat = pool.view(torch.uint8).view(pages * page, -1).clone()
        for j, l in enumerate(lists):
            slot = [int(table[j, r // page]) * page + r % page for r in range(lens[j])]
            old = flat.clone()
            for i in range(counts[j]):
                flat[slot[cached[j] + i]] = old[slot[cached[j] + l[i]]]
        want.append(flat)
    got = paged_kv_accept(pools[0], pools[1], table.cuda(), i32(cached), i32(acc.tolist()),
                          cu_seqlens_q=ph.cu_of(new).cuda())
    assert got.cpu().tolist() == [c + n for c, n in zip(cached, counts)]
    for p, w in zip(pools, want):
        assert torch.equal(p.view(torch.uint8).view(pages * page, -1).cpu(), w)
    assert_device_ok()


def test_accept_bad_tables_and_layouts():
    from fa4_ring import paged_kv_accept
    g = torch.Generator().manual_seed(3)
    pool = torch.randn(4, 16, 2, 128, generator=g).to(BF).cuda()
    table = i32([[0, -1, 99, -2 ** 31]])  # nodes on these pages cannot move
    before = pool.clone()
    lens = paged_kv_accept(pool, pool.clone(), table, i32([14]), i32([[1, 3, 20, 40]]), cu_seqlens_q=i32([0, 60]))
    assert lens.item() == 18
    want = before.clone()
    want[0, 14] = before[0, 15]
    assert torch.equal(pool, want)
    lens = paged_kv_accept(pool, pool.clone(), table[:, :1], i32([-9]), i32([[1, 30]]), cu_seqlens_q=i32([0, 60]))
    want[0, 0] = want[0, 1]
    assert lens.item() == 2 and torch.equal(pool, want)
    hf = before.transpose(1, 2).contiguous().transpose(1, 2)  # heads before rows
    paged_kv_accept(hf, hf.clone(), i32([[2, 1]]), i32([10]), i32([[2, 9]]), cu_seqlens_q=i32([0, 12]))
    want = before.clone()
    want[2, 10], want[2, 11] = before[2, 12], before[1, 3]
    assert torch.equal(hf, want)
    assert paged_kv_accept(pool, pool, table, i32([3]), torch.zeros(1, 0, dtype=torch.int32).cuda(),
                           cu_seqlens_q=i32([0, 4])).item() == 3
    assert_device_ok()


def test_refusals():
    from fa4_ring import paged_block_tables, paged_kv_accept, paged_kv_write
    pool = torch.zeros(4, 16, 2, 128, dtype=BF, device="cuda")
    k = torch.zeros(3, 2, 128, dtype=BF, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    for args, kw, err in (
            ((k.half(), k.half(), pool, pool, slots), {}, ValueError),          # another dtype
            ((k, k, pool, pool, slots), dict(k_descale=1.0), ValueError),       # descale of a copy
            ((k.float(), k.float(), pool, pool, slots), {}, ValueError),
            ((k[:, :1], k[:, :1], pool, pool, slots), {}, AssertionError),
            ((k, k, pool, pool, slots[:2]), {}, AssertionError),
            ((k.cpu(), k, pool, pool, slots), {}, RuntimeError),
            ((k, k, pool.transpose(2, 3), pool.transpose(2, 3), slots), {}, AssertionError),
            ((k[..., :4], k[..., :4], pool[..., :4], pool[..., :4], slots), {}, ValueError)):
        with pytest.raises(err):
            paged_kv_write(*args, **kw)
    one = i32([1])
    with pytest.raises(ValueError):
        paged_block_tables(one, one, one, page_size=16, num_tokens=1)            # no width
    with pytest.raises(AssertionError):
        paged_block_tables(one, i32([1, 1]), one, page_size=16, num_tokens=1, max_pages=2)
    with pytest.raises(AssertionError):
        paged_block_tables(one, one, one, page_size=0, num_tokens=1, max_pages=2)
    with pytest.raises(ValueError):
        paged_kv_accept(pool, pool, i32([[0]]), one, torch.zeros(1, 1025, dtype=torch.int32).cuda(),
                        cu_seqlens_q=i32([0, 1]))


@pytest.mark.parametrize("kv_dt", [BF, E4M3])
def test_serving_loop(kv_dt):
    """Prompt, then drafted trees step by step: plan, mask, write, attend, accept; the cache and
    the attention are those of a plain list of rows for each request."""
    from fa4_ring import (b200_attn_paged_tree, paged_block_tables, paged_kv_accept, paged_kv_write,
                          paged_tree_mask)
    g = torch.Generator().manual_seed(77)
    B, H, hk, D, page, width = 3, 8, 2, 128, 16, 24
    kd, vd = (0.02 + 0.01 * torch.rand(hk, generator=g) for _ in range(2))
    quant = kv_dt == E4M3
    desc = dict(k_descale=kd.cuda(), v_descale=vd.cuda()) if quant else {}
    pools = [torch.full((B * width, page, hk, D), math.nan).to(kv_dt).cuda() for _ in range(2)]
    free = torch.randperm(B * width, generator=g, dtype=torch.int32).cuda()
    table = None
    cached = i32([0] * B)
    rows = [[torch.zeros(0, hk, D, dtype=torch.float64)] * 2 for _ in range(B)]
    for step, new in enumerate(([50, 1, 17], [7, 9, 1], [1, 1, 1], [20, 0, 33], [12, 16, 5])):
        T = sum(new)
        k, v = (torch.randn(T, hk, D, generator=g).to(BF) for _ in range(2))
        q = torch.randn(T, H, D, generator=g).to(BF)
        plan = paged_block_tables(cached, i32(new), free, page_size=page, num_tokens=T + 2,
                                  block_table=table, max_pages=width)
        used, short = plan.pages.tolist()
        assert short == 0
        table, free = plan.block_table, free[used:]
        cu = plan.cu_seqlens_q
        tree = step > 0
        parents = ph.random_parents(new, g)
        mask = paged_tree_mask(parents.cuda(), cu, max_nodes=max(new)) if tree else None
        padded = [torch.cat([x, x[:2]]).cuda() for x in (k, v)]  # a padded batch: slots -1
        paged_kv_write(padded[0], padded[1], pools[0], pools[1], plan.slot_mapping, **desc)
        out = b200_attn_paged_tree(q.cuda(), pools[0], pools[1], table, cu_seqlens_q=cu,
                                   seq_lens=plan.seq_lens, max_seqlen_q=max(new), tree_mask=mask, **desc)
        cu = cu.cpu()
        seen = [ph.seen_of(parents, cu, j) for j in range(B)] if tree else None
        ends = [int(cu[j]) for j in range(B + 1)]
        ks = [torch.cat([rows[j][0], stored(k[ends[j]:ends[j + 1]], kd, kv_dt).double()]) for j in range(B)]
        vs = [torch.cat([rows[j][1], stored(v[ends[j]:ends[j + 1]], vd, kv_dt).double()]) for j in range(B)]
        # the plain cache as one page a request
        most = max(x.shape[0] for x in ks)
        flat = [torch.stack([torch.nn.functional.pad(x, (0, 0, 0, 0, 0, most - x.shape[0])) for x in xs]).to(kv_dt)
                for xs in (ks, vs)]
        lens = [x.shape[0] for x in ks]
        assert lens == plan.seq_lens.tolist()
        ph.check_attn(out, ph.attn(q, flat[0], flat[1], torch.arange(B)[:, None], cu, lens, seen,
                                   1 / math.sqrt(D), kd if quant else None, vd if quant else None))
        if not tree:
            cached = plan.seq_lens
            rows = [[ks[j], vs[j]] for j in range(B)]
            continue
        acc = torch.full((B, 6), -1, dtype=torch.int32)
        for j in range(B):
            if new[j] == 0:
                continue
            path = [int(torch.randint(new[j], (1,), generator=g))]
            while int(parents[ends[j] + path[0]]) >= 0:
                path.insert(0, int(parents[ends[j] + path[0]]))
            path = path[:6]
            acc[j, :len(path)] = torch.tensor(path, dtype=torch.int32)
            base = lens[j] - new[j]
            rows[j] = [torch.cat([x[:base], x[[base + a for a in path]]]) for x in (ks[j], vs[j])]
        cached = paged_kv_accept(pools[0], pools[1], table, cached, acc.cuda(), cu_seqlens_q=plan.cu_seqlens_q)
        assert cached.tolist() == [r[0].shape[0] for r in rows]
    assert_device_ok()


def test_write_descales_of_every_size():
    """The stored value is e4m3 of the fp32 quotient for any divisor: tiny, huge, negative, 0 and
    infinite ones, and subnormal ones."""
    from fa4_ring import paged_kv_write
    d = torch.tensor([0.0, math.inf, 1e-30, 1e30, 2.0 ** -60, -0.03, 1e-42, 3e38, 0.37, 2.0 ** 60])
    g = torch.Generator().manual_seed(7)
    x = torch.randn(40, 10, 64, generator=g) * torch.exp2(torch.randint(-11, 10, (40, 10, 64), generator=g).float())
    near = torch.where(torch.isfinite(d) & (d != 0), d, 1.0)
    x = (x.double() * near.double()[:, None]).to(BF)  # quotients over the whole of e4m3's range
    x[0, :, :5] = torch.tensor([0.0, math.inf, -math.inf, math.nan, 2.0 ** 127]).to(BF)
    pool = torch.zeros(3, 16, 10, 64, dtype=E4M3, device="cuda")
    other = torch.zeros_like(pool)
    paged_kv_write(x.cuda(), x.cuda(), pool, other, torch.arange(40).cuda(), k_descale=d.cuda(), v_descale=d.cuda())
    want = (x.float() / d[:, None]).clamp(-448, 448).to(E4M3).float()
    for p in (pool, other):
        got = p.view(48, 10, 64)[:40].float().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert_device_ok()


def test_write_rows_longer_than_a_block():
    from fa4_ring import paged_kv_write
    g = torch.Generator().manual_seed(11)
    for hk, D, T in ((20, 256, 9), (33, 64, 700), (7, 24, 3)):
        k, v = (torch.randn(T, hk, D, generator=g).to(F16).cuda() for _ in range(2))
        slots = torch.randperm(T + 13, generator=g)[:T].cuda()
        kp, vp = (torch.zeros(T + 13, 1, hk, D, dtype=F16, device="cuda") for _ in range(2))
        paged_kv_write(k, v, kp, vp, slots)
        assert torch.equal(kp[slots, 0], k) and torch.equal(vp[slots, 0], v)
        assert int((kp != 0).any(-1).any(-1).sum()) == T
    assert_device_ok()


def test_accept_in_empty_pools():
    from fa4_ring import paged_kv_accept
    pool = torch.zeros(0, 16, 2, 128, dtype=BF, device="cuda")
    lens = paged_kv_accept(pool, pool.clone(), i32([[-1], [-1]]), i32([4, 0]), i32([[1, 2], [0, 5]]),
                           cu_seqlens_q=i32([0, 6, 7]))
    assert lens.tolist() == [6, 1]


def test_two_steps_at_once():
    """Two requests sets, each written, planned and accepted on a stream of its own."""
    from fa4_ring import paged_kv_accept, paged_kv_write
    g = torch.Generator().manual_seed(13)
    sets = []
    for _ in range(2):
        pools = [torch.randn(64, 16, 4, 128, generator=g).to(BF) for _ in range(2)]
        rows = [torch.randn(96, 4, 128, generator=g).to(BF) for _ in range(2)]
        slots = torch.randperm(1024, generator=g)[:96]
        table = torch.randperm(64, generator=g)[:16].view(4, 4)
        acc = torch.tensor([[1, 3, 5, 9]] * 4)
        sets.append((pools, rows, slots, table, acc))

    def step(s, stream):
        (kp, vp), (k, v), slots, table, acc = s
        with torch.cuda.stream(stream):
            kp, vp = kp.cuda(), vp.cuda()
            k, v, slots = k.cuda(), v.cuda(), slots.cuda()
            table, acc = table.to(torch.int32).cuda(), acc.to(torch.int32).cuda()
            cached, cu = i32([20, 3, 40, 11]), i32([0, 12, 24, 36, 48])
            paged_kv_write(k, v, kp, vp, slots)
            lens = paged_kv_accept(kp, vp, table, cached, acc, cu_seqlens_q=cu)
        return kp, vp, lens

    one = [step(s, torch.cuda.current_stream()) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        both = [step(s, st) for s, st in zip(sets, streams)]
        torch.cuda.synchronize()
        for a, b in zip(one, both):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert_device_ok()
