"""Plain 64-bit forms of the paged-cache operators, for the tests (CPU, torch float64)."""

import math

import torch

E4M3 = torch.float8_e4m3fn
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def cu_of(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)


def random_parents(lens, g):
    """A random tree for each request: parents come before their children, -1 is a root."""
    return torch.cat([(torch.rand(n, generator=g) * (torch.arange(n) + 1)).floor().int() - 1
                      for n in lens] + [torch.zeros(0, dtype=torch.int32)])


def seen_of(parents, cu, j):
    """bool [n, n]: node i of request j sees node m."""
    a, n = int(cu[j]), int(cu[j + 1] - cu[j])
    seen = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        up = int(parents[a + i])
        if 0 <= up < i:
            seen[i] = seen[up]
        seen[i, i] = True
    return seen


def pack(seen, words):
    """bool [n, m] -> int64 [n, words]."""
    n, m = seen.shape
    bits = torch.zeros(n, words * 64, dtype=torch.int64)
    bits[:, :m] = seen.long()
    return (bits.view(n, words, 64) << torch.arange(64)).sum(-1)


def block_table(lens, page, g, spare=2, width=None):
    counts = [-(-n // page) for n in lens]
    perm = torch.randperm(sum(counts) + spare, generator=g, dtype=torch.int32)
    table = torch.full((len(lens), width or max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for j, c in enumerate(counts):
        table[j, :c] = perm[at:at + c]
        at += c
    return table, sum(counts) + spare


def rows_of(pool, table, j, n):
    """float64 [n, H_kv, D]: the first n cached rows of request j."""
    page = pool.shape[1]
    pos = torch.arange(n)
    pages = table[j, pos // page].long()
    return pool[pages, pos % page].double() if pool.dtype != E4M3 else \
        pool.view(torch.uint8)[pages, pos % page].view(E4M3).double()


def attn(q, k_pages, v_pages, table, cu, lens, seen, scale, kd=None, vd=None, qd=None):
    """(out, lse, tol, lse_tol) in float64; ``seen[j]`` bool [n, n] or None (causal).

    The tolerances follow the kernel's roundings.  Products of q and k are exact and summed in
    fp32, so a score errs by at most e = (D + 8) 2^-24 sum|q||k| scale (and a P by a factor
    1 + 2e, with 2^-20 for the hardware exponential); P is rounded once to the 16-bit operand
    type (half a step u_p relative, 2^-25 absolute for an f16 that is subnormal), O is summed
    in fp32, and out is rounded once (u_o).  Over an e4m3 cache P is an f16, and a bf16 q is
    two e4m3 terms of q 2^s with the row's largest in [2^7, 2^8): the first leaves at most half
    of its last place, the second holds that exactly but for what is below half of the least
    e4m3, 2^-10, so q errs by at most 2^-17 of the row's largest.  The descales and the
    scales of the operands add a few roundings in fp32.
    """
    T, H, D = q.shape
    hk = k_pages.shape[2]
    kv8 = k_pages.dtype == E4M3
    out_dt = torch.bfloat16 if q.dtype == E4M3 else q.dtype
    u_p = HALF_STEP[torch.float16 if kv8 else q.dtype]
    u_o = HALF_STEP[out_dt]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    one = torch.ones(hk, dtype=torch.float64)
    kd, vd, qd = (one if d is None else d.double().cpu() for d in (kd, vd, qd))
    for j in range(len(lens)):
        a, n, size = int(cu[j]), int(cu[j + 1] - cu[j]), int(lens[j])
        if n == 0 or size <= 0:
            continue
        k = rows_of(k_pages, table, j, size) * kd[:, None]
        v = rows_of(v_pages, table, j, size) * vd[:, None]
        node = torch.arange(size) - (size - n)
        vis = (node < 0)[None].expand(n, size).clone()
        s = torch.tril(torch.ones(n, n, dtype=torch.bool)) if seen is None else seen[j]
        new = node >= 0
        vis[:, new] = s[:, node[new]]
        for h in range(H):
            g = h // (H // hk)
            x = q[a:a + n, h].double() * qd[g]
            kk, vv = k[:, g], v[:, g]
            sc = torch.where(vis, x @ torch.nan_to_num(kk).T * scale, -math.inf)
            if not torch.isfinite(kk).all():  # only what is seen may be non-finite
                for i in range(n):
                    sc[i, vis[i]] = (kk[vis[i]] @ x[i]) * scale
            top = sc.amax(1, keepdim=True)
            p = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
            l = p.sum(1, keepdim=True)
            w = torch.where(l > 0, p / l, 0.0)
            for i in range(n):
                ii = vis[i]
                out[a + i, h] = w[i, ii] @ vv[ii]
                A = w[i, ii] @ vv[ii].abs()
                e = (D + 8) * 2.0 ** -24 * scale * float(
                    ((kk[ii].abs() @ x[i].abs()).max() if ii.any() else 0.0))
                if kv8 and q.dtype != E4M3:
                    e += 2.0 ** -17 * scale * float(x[i].abs().max()) * float(
                        kk[ii].abs().sum(1).max() if ii.any() else 0.0)
                m = int(ii.sum())
                rel = u_p + 2 * (2 * e + 2.0 ** -20) + (m + 8) * 2.0 ** -24
                low = m * 2.0 ** -25 * (vv[ii].abs().max(0).values if m else 0.0) \
                    if (kv8 or q.dtype == torch.float16) else 0.0
                tol[a + i, h] = rel * A + low + u_o * (A + out[a + i, h].abs()) + 2.0 ** -25
                ltol[a + i, h] = 2 * e + 2.0 ** -20 + m * 2.0 ** -24
            lse[a:a + n, h] = (top + torch.log(l))[:, 0]
    ltol += 2.0 ** -22 * torch.where(torch.isfinite(lse), lse.abs(), 0.0)
    return out, lse, tol, ltol


def check_attn(got, want, rows=None):
    (out, lse), (ro, rl, tol, ltol) = got, want
    out, lse = out.double().cpu(), lse.double().cpu()
    if rows is not None:
        out, lse, ro, rl, tol, ltol = (x[rows] for x in (out, lse, ro, rl, tol, ltol))
    fine = torch.isfinite(ro)
    assert torch.equal(torch.isfinite(out), fine), "finite where the formula is not, or the other way"
    over = ((out - ro).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (
        f"out off by {float((out - ro).abs()[fine].max()):.3e}, {float(over.max()):.3e} over its tolerance")
    same = torch.isfinite(rl)
    assert torch.equal(torch.isfinite(lse), same)
    assert torch.equal(lse[~same], rl[~same]) or rl[~same].isnan().any()
    lover = ((lse - rl).abs() - ltol)[same]
    assert lover.numel() == 0 or float(lover.max()) <= 0, f"lse {float(lover.max()):.3e} over its tolerance"
