"""Attention of decode steps and drafted trees over a paged cache (``b200_attn_paged_tree``)
against the 64-bit form of ``paged_helpers``, whose tolerances are derived there."""

import math

import pytest
import torch

import paged_helpers as ph
from gpu_helpers import assert_device_ok

pytestmark = pytest.mark.gpu

BF, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def make(lens, new, H, hk, D, q_dt, kv_dt, page, seed, tree=True, scale_q=1.0):
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    x = dict(lens=lens, new=new, cu=ph.cu_of(new), seen=None, mask=None, qd=None, kd=None, vd=None)

    def rand(shape, dt):
        r = torch.randn(shape, generator=g)
        return (r * 60).clamp(-448, 448).to(E4M3) if dt == E4M3 else r.to(dt)

    x["q"] = rand((T, H, D), q_dt) if q_dt == E4M3 else (rand((T, H, D), q_dt) * scale_q)
    x["table"], pages = ph.block_table(lens, page, g)
    x["k"], x["v"] = rand((pages, page, hk, D), kv_dt), rand((pages, page, hk, D), kv_dt)
    if q_dt == E4M3:
        x["qd"] = 0.01 + 0.01 * torch.rand(hk, generator=g)
    if kv_dt == E4M3:
        x["kd"], x["vd"] = (0.01 + 0.01 * torch.rand(hk, generator=g) for _ in range(2))
    if tree:
        parents = ph.random_parents(new, g)
        words = (max(max(new), 1) + 63) // 64
        x["seen"] = [ph.seen_of(parents, x["cu"], j) for j in range(len(new))]
        x["mask"] = torch.cat([ph.pack(s, words) for s in x["seen"]])
    return x


def want(x, scale=None):
    return ph.attn(x["q"], x["k"], x["v"], x["table"], x["cu"], x["lens"], x["seen"],
                   scale or 1.0 / math.sqrt(x["q"].shape[2]), x["kd"], x["vd"], x["qd"])


def dev(t):
    return None if t is None else t.cuda()


def call(x, q=None, k=None, v=None, **kw):
    from fa4_ring import b200_attn_paged_tree
    return b200_attn_paged_tree(
        dev(x["q"]) if q is None else q, dev(x["k"]) if k is None else k,
        dev(x["v"]) if v is None else v, dev(x["table"]), cu_seqlens_q=dev(x["cu"]),
        seq_lens=torch.tensor(x["lens"], dtype=torch.int32).cuda(),
        max_seqlen_q=max(x["new"] + [1]), tree_mask=dev(x["mask"]), q_descale=dev(x["qd"]),
        k_descale=dev(x["kd"]), v_descale=dev(x["vd"]), **kw)


LENS = [1, 300, 0, 127, 128, 129, 64, 513]
NEW = [1, 7, 0, 5, 1, 3, 64, 2]


@pytest.mark.parametrize("q_dt,kv_dt", [(BF, BF), (F16, F16), (BF, E4M3), (E4M3, E4M3)],
                         ids=["bf16", "f16", "bf16-e4m3", "e4m3"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (128, 128), (256, 32), (256, 256)])
def test_types_and_lengths(q_dt, kv_dt, D, page):
    x = make(LENS, NEW, 8, 2, D, q_dt, kv_dt, page, seed=D + page)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("H,hk", [(1, 1), (6, 2), (5, 1), (16, 1), (4, 4), (40, 2), (24, 8)])
def test_head_layouts(H, hk):
    x = make([200, 77], [9, 20], H, hk, 128, BF, BF, 32, seed=H * 10 + hk)
    ph.check_attn(call(x), want(x))
    x = make([200, 77], [1, 1], H, hk, 64, F16, F16, 16, seed=H * 10 + hk, tree=False)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("n,group", [(1, 1), (16, 8), (32, 4), (33, 4), (64, 8), (130, 3), (300, 1)])
def test_tree_sizes(n, group):
    """Rows that fill, just pass and span several 128-row tiles; masks of several words."""
    x = make([n, n + 257, n + 1000], [n, n, max(n // 2, 1)], 2 * group, 2, 128, BF, BF, 64, seed=n)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 300], [150, 128, 2]])
@pytest.mark.parametrize("kv_dt", [BF, E4M3])
def test_causal_without_a_mask(new, kv_dt):
    x = make([400, 1, 300], new if new[1] == 1 else [150, 1, 2], 8, 2, 128, BF, kv_dt, 64,
             seed=sum(new), tree=False)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


def test_more_new_tokens_than_cached_rows():
    """Bottom-right alignment: the first rows of a request that holds fewer rows see nothing."""
    from fa4_ring import b200_attn_paged_tree
    x = make([3], [3], 4, 1, 128, BF, BF, 16, seed=3, tree=False)
    q = torch.randn(5, 4, 128, generator=torch.Generator().manual_seed(9)).to(BF)
    out, lse = b200_attn_paged_tree(q.cuda(), dev(x["k"]), dev(x["v"]), dev(x["table"]),
                                    cu_seqlens_q=torch.tensor([0, 5], dtype=torch.int32).cuda(),
                                    seq_lens=torch.tensor([3], dtype=torch.int32).cuda(), max_seqlen_q=5)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == -math.inf).all())
    x["q"] = q[2:]
    ph.check_attn((out[2:], lse[2:]), want(x))


def test_long_cache_in_many_parts():
    """One request whose cache every SM takes a part of, beside short ones."""
    for kv_dt, D in ((BF, 128), (E4M3, 256), (F16, 64)):
        x = make([20011, 1, 40], [6, 1, 3], 4, 1, D, F16 if kv_dt == F16 else BF, kv_dt, 64, seed=5)
        ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("batch", [1, 147, 149, 700])
def test_many_short_requests(batch):
    lens = [1 + (7 * i) % 150 for i in range(batch)]
    x = make(lens, [1] * batch, 2, 1, 64, BF, BF, 16, seed=batch, tree=False)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("kv_dt", [BF, F16, E4M3])
def test_rows_that_see_nothing(kv_dt):
    """Mask rows of zeros: over an empty cache they see no key, over a cache only the cache."""
    x = make([4, 40, 130], [4, 4, 6], 4, 2, 64, F16 if kv_dt == F16 else BF, kv_dt, 16, seed=1)
    for j, i in ((0, 1), (0, 3), (1, 2), (2, 0)):
        x["seen"][j][i] = False
        x["mask"][int(x["cu"][j]) + i] = 0
    out, lse = call(x)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    ph.check_attn((out, lse), want(x))
    # a mask of ones in bits past the tree and past the cache adds nothing
    x["mask"][5] |= -(1 << 40)
    ph.check_attn(call(x), want(x))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kv_dt,D", [(BF, 128), (F16, 64), (E4M3, 128), (BF, 256), (E4M3, 256)])
def test_unseen_rows_may_hold_anything(bad, kv_dt, D):
    """Rows behind the cache, other requests' pages and siblings in the tree: NaN and infinities
    there do not reach a result; a row that sees one is not finite where the formula is not."""
    if kv_dt == E4M3 and not math.isnan(bad):
        pytest.skip("e4m3 has no infinities")
    lens, new = [130, 200, 33], [3, 9, 5]
    x = make(lens, new, 4, 2, D, F16 if kv_dt == F16 else BF, kv_dt, 64, seed=D)
    for name in ("k", "v"):
        pool = x[name].float()
        keep = torch.zeros(pool.shape[:2], dtype=torch.bool)
        for j, n in enumerate(lens):
            pos = torch.arange(n)
            keep[x["table"][j, pos // 64].long(), pos % 64] = True
        pool[~keep] = bad
        x[name] = pool.to(kv_dt)
    ph.check_attn(call(x), want(x))
    # node 4 of request 1 gets a bad value row: only the nodes that see it are touched
    r = 200 - 9 + 4
    pool = x["v"].float()
    pool[x["table"][1, r // 64].long(), r % 64] = bad
    x["v"] = pool.to(kv_dt)
    hit = x["seen"][1][:, 4]
    rows = torch.cat([torch.ones(3, dtype=torch.bool), ~hit, torch.ones(5, dtype=torch.bool)])
    got = call(x)
    ph.check_attn(got, want(x), rows)
    assert not torch.isfinite(got[0][~rows].float()).any()
    # and a bad key row
    x["v"] = torch.nan_to_num(x["v"].float(), 0.0, 0.0, 0.0).to(kv_dt)
    pool = x["k"].float()
    pool[x["table"][1, r // 64].long(), r % 64] = bad
    x["k"] = pool.to(kv_dt)
    ph.check_attn(call(x), want(x), rows)
    assert_device_ok()


def test_large_scores_and_scale():
    x = make([700, 90], [8, 8], 8, 2, 128, BF, BF, 64, seed=8, scale_q=40.0)
    ph.check_attn(call(x), want(x))
    ph.check_attn(call(x, softmax_scale=0.5), want(x, 0.5))
    # tiny, huge and zero queries against an e4m3 cache, and signs and zeros in the descales
    x = make([300], [4], 4, 1, 128, BF, E4M3, 64, seed=9)
    x["q"][0] *= 2.0 ** -30
    x["q"][1] *= 2.0 ** 17
    x["q"][2] = 0
    ph.check_attn(call(x, softmax_scale=2.0 ** -16), want(x, 2.0 ** -16))
    for kd, qd in ((-0.02, None), (0.0, None), (-0.015, 0.7), (0.01, -0.02)):
        q_dt = BF if qd is None else E4M3
        x = make([300, 5], [4, 2], 4, 1, 64, q_dt, E4M3, 64, seed=10)
        x["kd"] = torch.tensor([kd])
        x["qd"] = None if qd is None else torch.tensor([qd])
        ph.check_attn(call(x), want(x))


def test_queries_that_are_not_finite():
    """A non-finite query row is its own trouble: the rows beside it in the tile are right."""
    for kv_dt, D in ((BF, 128), (E4M3, 64), (E4M3, 256)):
        x = make([200, 30], [3, 4], 4, 2, D, BF, kv_dt, 32, seed=21)
        x["q"][1, 2, 5] = math.nan
        x["q"][4, 0, 0] = math.inf
        got = call(x)
        good = torch.ones(7, 4, dtype=torch.bool)
        good[1, 2] = good[4, 0] = False
        ref = want({**x, "q": torch.nan_to_num(x["q"], 0.0, 0.0, 0.0)})
        ph.check_attn(got, ref, good)
        assert not torch.isfinite(got[0].cpu()[~good].float()).any()


def test_rising_scores_rescale():
    """Scores that rise along the cache: the running maximum is replaced again and again."""
    x = make([900], [2], 2, 1, 64, F16, F16, 16, seed=4, tree=False)
    x["q"] = torch.ones_like(x["q"])
    pos = torch.arange(900)
    ramp = (pos.float() / 900 * 6)[:, None, None].expand(900, 1, 64).to(F16)
    x["k"][x["table"][0, pos // 16].long(), pos % 16] = ramp
    ph.check_attn(call(x), want(x))


def test_views_are_taken_as_they_are():
    """q cut out of a fused projection; pools as views of other layouts."""
    x = make([70, 300], [3, 6], 8, 2, 128, BF, BF, 32, seed=2)
    ref = call(x)
    fused = torch.randn(9, 8 * 128 + 512).to(BF).cuda()
    fused[:, :1024] = x["q"].reshape(9, -1).cuda()
    q = fused[:, :1024].view(9, 8, 128)
    assert not q.is_contiguous()
    odd = torch.randn(9, 8 * 128 + 3).to(BF).cuda()  # rows that are not 16-byte aligned
    odd[:, 3:] = x["q"].reshape(9, -1).cuda()
    heads_first = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3).cuda() for t in (x["k"], x["v"])]
    both = torch.stack([x["k"], x["v"]], 1).cuda()
    for kw in (dict(q=q), dict(q=odd[:, 3:].view(9, 8, 128)), dict(k=heads_first[0], v=heads_first[1]),
               dict(k=both[:, 0], v=both[:, 1])):
        got = call(x, **kw)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    with pytest.raises(ValueError):  # a pool is never copied
        call(x, k=both[:, 0].transpose(2, 3).contiguous().transpose(2, 3), v=both[:, 1])
    assert_device_ok()


def test_pages_past_32_bit_offsets():
    x = make([200, 50], [4, 4], 8, 8, 128, BF, BF, 128, seed=6)
    pages = 2 ** 32 // (128 * 8 * 128) + 9  # the last pages start past 2^32 elements
    ref = call(x)
    big = torch.zeros(2, pages, 128, 8, 128, dtype=BF, device="cuda")
    n = x["k"].shape[0]
    big[0, pages - n:], big[1, pages - n:] = x["k"].cuda(), x["v"].cuda()
    x["table"] = torch.where(x["table"] < 0, -1, x["table"] + pages - n)
    got = call(x, k=big[0], v=big[1])
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert_device_ok()


def test_bad_pages_read_zeros():
    """A page outside the pool counts as rows of zeros, as in b200_attn_paged."""
    x = make([100], [2], 4, 1, 128, BF, BF, 16, seed=7, tree=False)
    y = {**x, "k": x["k"].clone(), "v": x["v"].clone(), "table": x["table"].clone()}
    for e, bad in ((1, -1), (3, 10 ** 6), (4, -2 ** 31)):
        page = int(x["table"][0, e])
        y["k"][page] = 0
        y["v"][page] = 0
        x["table"][0, e] = bad
    ph.check_attn(call(x), want(y))
    # a table narrower than the cache: the rows behind it, the new ones here, do not exist
    x["table"], x["k"], x["v"] = y["table"][:, :5], y["k"], y["v"]
    z = {**y, "lens": [82], "seen": [torch.zeros(2, 2, dtype=torch.bool)]}
    ph.check_attn(call(x), want(z))
    assert_device_ok()


def _raw(x, out, lse, ws, cu=None, lens=None):
    from fa4_ring import _lib
    from fa4_ring.attn_backend import pool_strides
    k, v, q = dev(x["k"]), dev(x["v"]), dev(x["q"])
    tb, mask = dev(x["table"]), dev(x["mask"])
    cu = dev(x["cu"]) if cu is None else cu
    lens = torch.tensor(x["lens"], dtype=torch.int32).cuda() if lens is None else lens
    T, H, D = q.shape
    rc = _lib.load().fa4cp_attn_fwd_paged_tree(
        q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), pool_strides(k, "k"),
        pool_strides(v, "v"), tb.data_ptr(), k.shape[1], k.shape[0], tb.shape[1], out.data_ptr(),
        lse.data_ptr(), cu.data_ptr(), lens.data_ptr(), cu.numel() - 1, max(x["new"]), T, H,
        k.shape[2], D, _lib.dtype_code(q.dtype), _lib.dtype_code(k.dtype), _lib.ptr(mask),
        0 if mask is None else mask.shape[1], 1.0 / math.sqrt(D), None, None, None, ws.data_ptr(),
        ws.numel(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc


def test_rows_behind_the_last_request_are_left():
    """A padded batch: q, out and lse hold more rows than cu_seqlens_q describes, some requests
    are idle; only the described rows are written."""
    from fa4_ring import _lib
    x = make([50, 0, 300], [4, 0, 9], 8, 2, 128, BF, BF, 16, seed=12)
    ref = call(x)
    pad = 5
    x["q"] = torch.cat([x["q"], torch.full((pad, 8, 128), math.nan).to(BF)])
    x["mask"] = torch.cat([x["mask"], torch.full((pad, 1), -1)])
    out = torch.full((13 + pad, 8, 128), 7.0, dtype=BF, device="cuda")
    lse = torch.full((13 + pad, 8), 7.0, device="cuda")
    n = _lib.load().fa4cp_attn_paged_tree_workspace_bytes(8, 2, 128, 9)
    ws = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")  # NaNs, and a guard
    assert _raw(x, out, lse, ws[:n]) == 0
    assert torch.equal(out[:13], ref[0]) and torch.equal(lse[:13], ref[1])
    assert bool((out[13:] == 7).all()) and bool((lse[13:] == 7).all())
    assert bool((ws[n:] == 255).all())
    # idle requests of negative length, and no request at all
    cu = torch.tensor([0, 4, 4, 4], dtype=torch.int32).cuda()
    out.fill_(7.0)
    assert _raw(x, out, lse, ws[:n], cu, torch.tensor([50, -3, -1], dtype=torch.int32).cuda()) == 0
    assert torch.equal(out[:4], ref[0][:4]) and bool((out[4:] == 7).all())
    if n > 16:
        assert _raw(x, out, lse, ws[:n - 16]) == -1
    assert_device_ok()


def test_streams_and_graphs():
    """Another stream; a captured step replayed with other lengths; two graphs that share the
    allocator's pool replayed in turn."""
    from fa4_ring import b200_attn_paged_tree
    x = make([900, 300], [4, 4], 8, 2, 128, BF, BF, 64, seed=13)
    y = {**x, "lens": [700, 290]}
    want_x, want_y = want(x), want(y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(x)
    side.synchronize()
    ph.check_attn(got, want_x)
    q, k, v, tb, cu, mask = (dev(x[n]) for n in ("q", "k", "v", "table", "cu", "mask"))
    lens = torch.tensor(x["lens"], dtype=torch.int32).cuda()

    def step():
        return b200_attn_paged_tree(q, k, v, tb, cu_seqlens_q=cu, seq_lens=lens, max_seqlen_q=4,
                                    tree_mask=mask)
    step()
    graphs, outs, pool = [], [], None
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            outs.append(step())
        pool = gr.pool()
        graphs.append(gr)
    for i in (0, 1, 0):
        lens.copy_(torch.tensor(x["lens"] if i == 0 else y["lens"], dtype=torch.int32))
        graphs[i].replay()
        torch.cuda.synchronize()
        ph.check_attn(outs[i], want_x if i == 0 else want_y)
    assert_device_ok()


def test_same_call_gives_the_same_bits():
    x = make([5000, 800, 33], [12, 3, 9], 8, 2, 128, BF, E4M3, 64, seed=14)
    a = call(x)
    for _ in range(3):
        b = call(x)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_agrees_with_paged_prefill_attention():
    """One token a request is the last row of b200_attn_paged over the same pages."""
    from fa4_ring.attn_backend import b200_attn_paged
    x = make([1000, 129], [1, 1], 8, 2, 128, BF, BF, 128, seed=15, tree=False)
    out, lse = call(x)
    o2, l2 = b200_attn_paged(dev(x["q"]), dev(x["k"]), dev(x["v"]), dev(x["table"]),
                             cu_seqlens_q=dev(x["cu"]), cu_seqlens_k=ph.cu_of(x["lens"]).cuda(),
                             max_seqlen_q=1, causal=True)
    w = want(x)
    ph.check_attn((o2, l2), w)
    ph.check_attn((out, lse), w)


@pytest.mark.parametrize("n,group,D,kv_dt", [(33, 4, 128, E4M3), (64, 8, 64, E4M3), (130, 3, 256, E4M3), (3, 160, 128, BF),
                                             (1, 300, 64, F16), (2, 129, 256, E4M3)])
def test_several_row_tiles(n, group, D, kv_dt):
    """More rows than a tile holds: many tokens, or more query heads of one K/V head than that."""
    q_dt = F16 if kv_dt == F16 else BF
    x = make([n, n + 300, n + 77], [n, max(n // 2, 1), n], group, 1, D, q_dt, kv_dt, 32, seed=n + group)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


@pytest.mark.parametrize("kv_dt,D", [(BF, 128), (E4M3, 64), (E4M3, 256)])
def test_many_row_tiles_of_a_block(kv_dt, D):
    """Some 20 short row tiles for every SM: the ring in which the items are passed on wraps."""
    lens = [1 + (11 * i) % 90 for i in range(750)]
    x = make(lens, [1] * 750, 4, 4, D, BF, kv_dt, 16, seed=D, tree=False)
    ph.check_attn(call(x), want(x))
    assert_device_ok()


def test_requests_that_share_pages():
    """A prefix held once: the first pages of two requests are the same."""
    x = make([200, 200], [5, 3], 8, 2, 128, BF, BF, 32, seed=16)
    x["table"][1, :5] = x["table"][0, :5]
    ph.check_attn(call(x), want(x))


def test_two_calls_at_once():
    from fa4_ring import b200_attn_paged_tree
    xs = [make([3000, 40, 700], [7, 1, 12], 8, 2, 128, BF, kv_dt, 64, seed=17) for kv_dt in (BF, E4M3)]
    one = [call(x) for x in xs]
    args = []
    for x in xs:
        args.append(((dev(x["q"]), dev(x["k"]), dev(x["v"]), dev(x["table"])), dict(
            cu_seqlens_q=dev(x["cu"]), seq_lens=torch.tensor(x["lens"], dtype=torch.int32).cuda(),
            max_seqlen_q=12, tree_mask=dev(x["mask"]), k_descale=dev(x["kd"]), v_descale=dev(x["vd"]))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        both = []
        for (a, kw), st in zip(args, streams):
            with torch.cuda.stream(st):
                both.append(b200_attn_paged_tree(*a, **kw))
        torch.cuda.synchronize()
        for a, b in zip(one, both):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert_device_ok()


def test_refusals():
    x = make([40], [2], 4, 2, 128, BF, BF, 16, seed=16)
    for change, err in ((dict(page=24), ValueError), (dict(d=96), NotImplementedError)):
        y = make([40], [2], 4, 2, change.get("d", 128), BF, BF, change.get("page", 16), seed=16)
        with pytest.raises(err):
            call(y)
    with pytest.raises(ValueError):
        call({**x, "kd": torch.ones(2)})          # descales without e4m3
    with pytest.raises(ValueError):
        call(x, softmax_scale=0.0)
    with pytest.raises(ValueError):
        call({**x, "q": x["q"].to(F16)})          # q and the pools differ
    with pytest.raises(AssertionError):
        call({**x, "mask": x["mask"][:1]})
    with pytest.raises(AssertionError):
        call({**x, "q": x["q"][:, :3]})           # 3 heads over 2
    with pytest.raises(RuntimeError, match="CUDA"):
        call(x, q=x["q"])
