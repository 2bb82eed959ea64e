"""Edges of the paged-cache operators: partly filled warps, hidden rows, unaligned views, bounds that
run past the tensors."""

import math

import pytest
import torch

import paged_helpers as ph
from gpu_helpers import assert_device_ok
from test_gpu_paged_tree import call, dev, make, want

pytestmark = pytest.mark.gpu

BF, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("kv_dt", [BF, F16, E4M3])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 31, 33, 65, 97])
def test_partly_filled_warps(kv_dt, D, rows):
    """A row tile that ends inside a warp, whole and in parts: its rows, and only those, come out."""
    q_dt = F16 if kv_dt == F16 else BF
    x = make([90, rows + 3000], [rows, rows], 1, 1, D, q_dt, kv_dt, 32, seed=rows + D)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kv_dt,D", [(BF, 128), (F16, 64), (E4M3, 128), (BF, 256), (E4M3, 256)])
def test_one_token_that_does_not_see_itself(kv_dt, D, bad):
    """A request of one token whose mask hides the token's own row: whatever the row holds stays out,
    over a cache and over none."""
    if kv_dt == E4M3 and not math.isnan(bad):
        pytest.skip("e4m3 has no infinities")
    x = make([1, 70, 1300], [1, 1, 1], 4, 2, D, F16 if kv_dt == F16 else BF, kv_dt, 16, seed=D)
    for j, n in enumerate(x["lens"]):
        x["seen"][j][0] = False
        x["mask"][j] = 0
        page = int(x["table"][j, (n - 1) // 16])
        for name in ("k", "v"):
            pool = x[name].float()
            pool[page, (n - 1) % 16] = bad
            x[name] = pool.to(kv_dt)
    out, lse = call(x)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    ph.check_attn((out, lse), want(x))
    # a mask that shows the row again
    x["seen"][1][0] = True
    x["mask"][1] = 1
    out, lse = call(x)
    assert not torch.isfinite(out[1].float()).any()
    ph.check_attn((out, lse), want(x), torch.tensor([True, False, True]))
    assert_device_ok()


@pytest.mark.parametrize("q_dt,kv_dt", [(F16, F16), (BF, E4M3), (E4M3, E4M3)], ids=["f16", "bf16-e4m3", "e4m3"])
@pytest.mark.parametrize("D,gap", [(64, 16), (64, 18), (64, 20), (128, 18), (256, 18)])
def test_weights_far_below_the_largest(q_dt, kv_dt, D, gap):
    """A few keys `gap` above all others, with values of 0: the others make the result.

    P is an f16 with its largest at 2^7 or more, so a weight is off by at most half of f16's least
    value, 2^-25, of 2^7 of the largest: m 2^-32 in all, beside the relative errors that
    paged_helpers.attn derives.  (Only the keys of one CTA share a largest P, so there are as many
    requests as two for each CTA, over the same pages.)"""
    from fa4_ring import b200_attn_paged_tree
    n, page, batch = 16384, 128, 296
    scale = 1.0 / D
    top = torch.tensor(gap / 4.0)  # q = 4, K = gap / 4: a score of gap; both are e4m3 values
    assert float(top.to(E4M3)) == float(top)
    k, v = torch.zeros(n, 1, D), torch.ones(n, 1, D)
    strong = torch.arange(0, 256, 32)  # of either warpgroup's tiles
    k[strong], v[strong] = top, 0.0
    q = torch.full((batch, 4, D), 4.0)
    k, v = (t.view(n // page, page, 1, D).to(kv_dt).cuda() for t in (k, v))
    table = torch.arange(n // page, dtype=torch.int32).expand(batch, -1).contiguous().cuda()
    out, lse = b200_attn_paged_tree(
        q.to(q_dt).cuda(), k, v, table, cu_seqlens_q=torch.arange(batch + 1, dtype=torch.int32).cuda(),
        seq_lens=torch.full((batch,), n, dtype=torch.int32).cuda(), max_seqlen_q=1, softmax_scale=scale)
    rest, few = n - len(strong), len(strong)
    total = few + rest * math.exp(-gap)
    exact = rest * math.exp(-gap) / total
    e = (D + 8) * 2.0 ** -24 * gap
    if kv_dt == E4M3 and q_dt != E4M3:
        e += 2.0 ** -17 * scale * 4.0 * D * gap / 4.0
    rel = 2.0 ** -11 + 2 * (2 * e + 2.0 ** -20) + (n + 8) * 2.0 ** -24
    u_o = 2.0 ** -11 if q_dt == F16 else 2.0 ** -8
    tol = rel * exact + n * 2.0 ** -32 + 2 * u_o * exact + 2.0 ** -25
    err = (out.double() - exact).abs().max().item()
    assert err <= tol, f"off by {err:.3e} of {exact:.3e}, allowed {tol:.3e}"
    want_lse = gap + math.log(total)
    err = (lse.double() - want_lse).abs().max().item()
    assert err <= 2 * e + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -22 * want_lse
    assert_device_ok()


@pytest.mark.parametrize("q_dt,kv_dt", [(F16, F16), (BF, BF)])
@pytest.mark.parametrize("D,tile", [(64, 64), (128, 64), (256, 32)])
def test_scores_past_the_steps_of_32_bits(q_dt, kv_dt, D, tile):
    """Scores of 2^26 in log2 units, where fp32 counts in steps of 4 and 8: the second half of the
    keys is 8 above the first, the most by which a maximum is left as it is.  The scores and their
    differences are exact, so the weights 1 and 256 are."""
    from fa4_ring import b200_attn_paged_tree
    n, batch = 4 * tile, 444  # as many requests as give a CTA whole ones
    k = torch.zeros(n, 1, D)
    k[:, 0, 0] = 4096.0
    k[n // 2:, 0, 1] = 2.0
    v = torch.zeros(n, 1, D)
    v[n // 2:, 0, ::2] = 1.0
    v[:n // 2, 0, 1::2] = 1.0
    q = torch.zeros(batch, 1, D)
    q[:, 0, 0], q[:, 0, 1] = 4096.0, 1.0
    table = torch.arange(n // 32, dtype=torch.int32).expand(batch, -1).contiguous().cuda()
    out, lse = b200_attn_paged_tree(
        q.to(q_dt).cuda(), k.view(-1, 32, 1, D).to(kv_dt).cuda(), v.view(-1, 32, 1, D).to(kv_dt).cuda(), table,
        cu_seqlens_q=torch.arange(batch + 1, dtype=torch.int32).cuda(),
        seq_lens=torch.full((batch,), n, dtype=torch.int32).cuda(), max_seqlen_q=1, softmax_scale=4 * math.log(2))
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    # the weights are powers of two (exact in P), the hardware exponential is good to 2^-20, the scale to
    # 2^-23 of 8, and the result is rounded once
    for part, exact in ((out[..., ::2], 256 / 257), (out[..., 1::2], 1 / 257)):
        tol = exact * (ph.HALF_STEP[q_dt] + 2.0 ** -18)
        assert (part.double() - exact).abs().max().item() <= tol
    assert_device_ok()


def test_unaligned_rows_of_one_token():
    """One token at an address that is not 16-byte aligned, dense as it is, is copied like any other
    view: a slice of a fused projection, and rows at an odd offset of a flat buffer."""
    from fa4_ring import paged_kv_write
    for new in ([1], [1, 4]):
        T = sum(new)
        x = make([70 + n for n in new], new, 8, 2, 128, BF, BF, 32, seed=31, tree=False)
        ref = call(x)
        odd = torch.zeros(T, 8 * 128 + 3, dtype=BF, device="cuda")
        odd[:, 3:] = x["q"].reshape(T, -1).cuda()
        flat = torch.zeros(1 + T * 8 * 128, dtype=BF, device="cuda")
        flat[1:] = x["q"].reshape(-1).cuda()
        for q in (odd[:, 3:].view(T, 8, 128), flat[1:].view(T, 8, 128)):
            assert q.data_ptr() % 16
            got = call(x, q=q)
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        slots = torch.arange(T).cuda() + 5
        rows = torch.randn(2, T, 2, 128, generator=torch.Generator().manual_seed(3)).to(BF).cuda()
        wide = torch.zeros(T, 1 + 512, dtype=BF, device="cuda")
        wide[:, 1:] = rows.permute(1, 0, 2, 3).reshape(T, 512)
        k, v = (wide[:, 1 + 256 * i:257 + 256 * i].view(T, 2, 128) for i in (0, 1))
        pools = torch.zeros(2, 2, 16, 2, 128, dtype=BF, device="cuda")
        paged_kv_write(k, v, pools[0], pools[1], slots)
        assert torch.equal(pools.view(2, 32, 2, 128)[:, 5:5 + T], rows)
    assert_device_ok()


@pytest.mark.parametrize("cu,total", [([0, 4, 14], 10), ([0, 14], 10), ([-3, 2, 6], 9), ([12, 14], 10),
                                      ([-9, -2], 5), ([0, 3, 3, 8, 2 ** 31 - 1], 11), ([-2 ** 31, 2, 5], 7)])
@pytest.mark.parametrize("nodes", [16, 130])
def test_tree_mask_bounds_past_the_rows(cu, total, nodes):
    """A tree whose bounds leave the rows is no tree: its rows are 0, as those outside every tree,
    and the trees beside it are whole."""
    from fa4_ring import _lib
    words = (nodes + 63) // 64
    parents = torch.tensor([(i % 3) - 1 for i in range(total)], dtype=torch.int32)
    mask = torch.full((total + 2, words), -1, dtype=torch.int64, device="cuda")
    par, bounds = parents.cuda(), i32(cu)
    rc = _lib.load().fa4cp_paged_tree_mask(par.data_ptr(), bounds.data_ptr(), len(cu) - 1, total, nodes,
                                           mask.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0
    want_mask = torch.zeros(total, words, dtype=torch.int64)
    for j, (a, b) in enumerate(zip(cu, cu[1:])):
        if 0 <= a < b <= total:
            want_mask[a:b] = ph.pack(ph.seen_of(parents, cu, j), words)
    assert torch.equal(mask[:total].cpu(), want_mask)
    assert bool((mask[total:] == -1).all())


@pytest.mark.parametrize("number", [0.02, torch.tensor(0.02), torch.tensor([[0.02]]), torch.tensor([0.02])],
                         ids=["float", "0-d", "1x1", "1"])
def test_capture_with_descales_on_the_host(number):
    """A descale that is one number, wherever it is, is no copy from the host: the calls can be
    captured into a graph, and give what a descale on the device gives."""
    from fa4_ring import b200_attn_paged_tree, paged_kv_write
    x = make([40, 9], [2, 1], 4, 1, 128, BF, E4M3, 16, seed=41, tree=False)
    x["kd"] = x["vd"] = torch.tensor([0.02])
    ref = call(x)
    q, k, v, tb, cu = (dev(x[n]) for n in ("q", "k", "v", "table", "cu"))
    lens = i32(x["lens"])
    rows = torch.randn(3, 1, 128, generator=torch.Generator().manual_seed(2)).to(BF).cuda()
    slots = torch.tensor([1, 5, 17]).cuda()
    pools = torch.zeros(4, 2, 16, 1, 128, dtype=E4M3, device="cuda")
    paged_kv_write(rows, rows, pools[0], pools[1], slots, k_descale=dev(x["kd"]), v_descale=dev(x["kd"]))

    def step():
        paged_kv_write(rows, rows, pools[2], pools[3], slots, k_descale=number, v_descale=number)
        return b200_attn_paged_tree(q, k, v, tb, cu_seqlens_q=cu, seq_lens=lens, max_seqlen_q=2,
                                    k_descale=number, v_descale=number)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = step()
    pools.view(torch.uint8)[2:] = 0
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    assert torch.equal(pools[2].view(torch.uint8), pools[0].view(torch.uint8))
    assert torch.equal(pools[3].view(torch.uint8), pools[1].view(torch.uint8))
    assert_device_ok()


def test_launches_counted():
    """The attention is two kernels: the parts, and their join."""
    from fa4_ring import _lib
    x = make([40], [2], 4, 1, 128, BF, BF, 16, seed=44)
    before = _lib.launch_count
    call(x)
    assert _lib.launch_count == before + 2


@pytest.mark.parametrize("q_dt,kv_dt,D,page", [(BF, BF, 64, 256), (BF, E4M3, 128, 128), (F16, F16, 256, 512)])
@pytest.mark.parametrize("shown", [False, True])
def test_a_cache_that_ends_at_the_last_int32(q_dt, kv_dt, D, page, shown):
    """2^31 - 1 cached rows, over a table that names one page again and again: the last tile ends
    where 32 bits do.  The row behind the cache holds NaN, and so does, if it is shown, the last of two
    new rows."""
    from fa4_ring import b200_attn_paged_tree
    n = 2 ** 31 - 1
    table = torch.zeros(1, 2 ** 31 // page, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    k = torch.zeros(2, page, 1, D)
    v = torch.ones(2, page, 1, D)
    k[1, page - 1], v[1, page - 1] = math.nan, math.nan  # row 2^31 - 1
    if shown:
        v[1, page - 2] = math.nan                         # row 2^31 - 2: the second new row
    q = torch.ones(2, 1, D)
    out, lse = b200_attn_paged_tree(q.to(q_dt).cuda(), k.to(kv_dt).cuda(), v.to(kv_dt).cuda(), table,
                                    cu_seqlens_q=i32([0, 2]), seq_lens=i32([n]), max_seqlen_q=2)
    # all weights are one power of two, so the sums and O are exact until the parts are joined
    good = out if not shown else out[:1]
    assert ((good.double() - 1).abs() <= ph.HALF_STEP[q_dt] + 2.0 ** -15).all()
    assert not shown or out[1].isnan().all()
    assert (lse.double() - math.log(n)).abs().max().item() <= 2.0 ** -20 + 2.0 ** -22 * math.log(n) + 2.0 ** -16
    assert_device_ok()


@pytest.mark.parametrize("kv_dt", [BF, E4M3])
def test_a_whole_step_captured(kv_dt):
    """Plan, mask, write, attention and accept as one graph, replayed with other lengths, trees and
    paths (requests of no tokens and of one among them): what the calls give one by one."""
    from fa4_ring import (b200_attn_paged_tree, paged_block_tables, paged_kv_accept, paged_kv_write,
                          paged_tree_mask)
    g = torch.Generator().manual_seed(51)
    B, H, hk, D, page, width, T = 3, 8, 2, 128, 16, 20, 24
    desc = dict(k_descale=0.02, v_descale=torch.tensor(0.02)) if kv_dt == E4M3 else {}
    table = torch.randperm(B * width, generator=g, dtype=torch.int32).view(B, width).clone()
    table[:, 15:] = -1
    owned = set(table[:, :15].flatten().tolist())
    free = [p for p in range(B * width) if p not in owned]
    fixed = dict(table=table.cuda(), free=i32(free))
    state = dict(cached=i32([0] * B), new=i32([0] * B), parents=i32([0] * T), accepted=i32([[-1] * 4] * B))
    pools0 = [(torch.randn(B * width, page, hk, D, generator=g) * 40).to(kv_dt).cuda() for _ in range(2)]
    x = [torch.randn(T, h, D, generator=g).to(BF).cuda() for h in (H, hk, hk)]

    def step(pools):
        plan = paged_block_tables(state["cached"], state["new"], fixed["free"], page_size=page, num_tokens=T,
                                  block_table=fixed["table"])
        mask = paged_tree_mask(state["parents"], plan.cu_seqlens_q, max_nodes=T)
        paged_kv_write(x[1], x[2], pools[0], pools[1], plan.slot_mapping, **desc)
        out, lse = b200_attn_paged_tree(x[0], pools[0], pools[1], plan.block_table, cu_seqlens_q=plan.cu_seqlens_q,
                                        seq_lens=plan.seq_lens, max_seqlen_q=T, tree_mask=mask, **desc)
        lens = paged_kv_accept(pools[0], pools[1], plan.block_table, state["cached"], state["accepted"],
                               cu_seqlens_q=plan.cu_seqlens_q)
        return plan, mask, out, lse, lens

    ours = [p.clone() for p in pools0]
    step(ours)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step(ours)
    for cached, new in (([230, 7, 100], [12, 1, 11]), ([0, 239, 240], [1, 0, 9]), ([64, 1, 3], [8, 8, 8])):
        state["cached"].copy_(i32(cached))
        state["new"].copy_(i32(new))
        par = ph.random_parents(new, g)
        state["parents"].fill_(-1)
        state["parents"][:par.numel()].copy_(par)
        state["accepted"].copy_(torch.randint(-1, 9, (B, 4), generator=g).sort(1).values.int())
        for p, q in zip(ours, pools0):
            p.view(torch.uint8).copy_(q.view(torch.uint8))
        gr.replay()
        torch.cuda.synchronize()
        theirs = [p.clone() for p in pools0]
        want_step = step(theirs)
        n = sum(new)
        for a, b in zip(got[0], want_step[0]):
            assert torch.equal(a, b)
        assert torch.equal(got[1], want_step[1]) and torch.equal(got[4], want_step[4])
        assert torch.equal(got[2][:n], want_step[2][:n]) and torch.equal(got[3][:n], want_step[3][:n])
        for a, b in zip(ours, theirs):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert_device_ok()
