"""Per-chunk attention on B200 (replaces ``fa4_ring/fa4_backend.py:58-123``).

``b200_attn`` has the calling convention of the reference's ``fa4_attn``: 3-D varlen
``[total, H, D]`` tensors plus ``cu_seqlens_q/k`` and ``max_seqlen_q/k``, optional
FP8 descales, and returns ``(out[Tq, H, D], lse[Tq, H])`` with LSE in float32 natural
log, already in the ``[T, H]`` layout the mergers use (no transpose copy).  It runs
the hand-written sm_100a kernel of ``fa4cp_attn_fwd`` (tcgen05 MMA, TMEM
accumulators, TMA tiles); FP8 e4m3 inputs produce a bf16 output.

``attn_into`` is the lower-level entry the ring uses: it writes (or, with
``accumulate=True``, merges) a step's partial into caller-owned ``out``/``lse`` for
one of the three zig-zag step patterns, addressing the row halves in place.
"""

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch

from . import _lib

PATTERN_VARLEN = _lib.PATTERN_VARLEN
PATTERN_FRONT_KV = _lib.PATTERN_FRONT_KV
PATTERN_BACK_Q = _lib.PATTERN_BACK_Q

SUPPORTED_HEAD_DIMS = {torch.bfloat16: (64, 128, 256), torch.float16: (64, 128, 256),
                       torch.float8_e4m3fn: (128,)}
# bf16 query with e4m3 K/V (K/V dequantised to bf16 in a workspace, then the bf16 kernel)
MIXED_HEAD_DIMS = (64, 128, 256)


def is_mixed(q: torch.Tensor, k: torch.Tensor) -> bool:
    return q.dtype == torch.bfloat16 and k.dtype == torch.float8_e4m3fn


def has_backend() -> bool:
    """True when the CUDA library loads (the reference's ``has_fa4``, fa4_backend.py:41-42)."""
    try:
        _lib.load()
        return True
    except RuntimeError:
        return False


def norm_descale(d: Optional[torch.Tensor], h_kv: int, device) -> Optional[torch.Tensor]:
    """Normalise an FP8 descale (scalar, ``[H_kv]`` or ``(1, H_kv)``) to a contiguous fp32
    ``[H_kv]`` CUDA tensor (fa4_ring/fa4_backend.py:45-55)."""
    if d is None:
        return None
    if (torch.is_tensor(d) and d.dtype is torch.float32 and d.dim() == 1 and d.numel() == h_kv
            and d.device == device and d.is_contiguous()):
        return d
    if not torch.is_tensor(d):
        return torch.full((h_kv,), float(d), dtype=torch.float32, device=device)
    if not d.is_cuda and (d.dim() == 0 or d.numel() == h_kv == 1):
        # one number on the host is filled in on the device: a copy of it would wait for the
        # stream, and could not be captured into a graph
        return torch.full((h_kv,), d.detach().item(), dtype=torch.float32, device=device)
    d = d.to(device=device, dtype=torch.float32)
    if d.dim() == 0:
        d = d.reshape(1).expand(h_kv)
    elif d.dim() == 2:
        d = d.reshape(-1)
    assert d.numel() == h_kv, f"descale must have H_kv={h_kv} entries, got {d.numel()}"
    return d.contiguous()


def out_dtype_for(dt: torch.dtype) -> torch.dtype:
    return torch.bfloat16 if dt == torch.float8_e4m3fn else dt


def _check_qkv(q, k, v):
    _lib.require_cuda(q, k, v)
    assert q.dim() == 3 and k.dim() == 3 and v.dim() == 3, "expected [T, H, D] tensors"
    assert k.dtype == v.dtype, "k and v must share a dtype"
    assert q.dtype == k.dtype or is_mixed(q, k), (
        "q, k, v must share a dtype (or bf16 q with e4m3 k/v)")
    assert k.shape == v.shape, "k and v must have the same shape"
    assert q.shape[2] == k.shape[2], "q and k head_dim differ"
    H, Hkv, D = q.shape[1], k.shape[1], q.shape[2]
    assert H % Hkv == 0, f"H_q={H} not a multiple of H_kv={Hkv}"
    if is_mixed(q, k):
        if D not in MIXED_HEAD_DIMS:
            raise NotImplementedError(f"head_dim {D} is not supported for bf16 q x e4m3 kv")
    elif q.dtype not in SUPPORTED_HEAD_DIMS or D not in SUPPORTED_HEAD_DIMS[q.dtype]:
        raise NotImplementedError(f"head_dim {D} with dtype {q.dtype} is not supported")


# Optional per-launch timing: when set to a list, every attn_into launch appends
# (start_event, end_event, pattern) recorded on the launching stream.
launch_timer = None


def attn_into(q, k, v, out, lse, cu_q, cu_k, *, nseq: int, max_seqlen_q: int, pattern: int,
              causal: bool, softmax_scale: float, q_descale=None, k_descale=None,
              v_descale=None, accumulate: bool = False) -> None:
    """Launch ``fa4cp_attn_fwd`` on the current stream.  All tensors contiguous CUDA."""
    lib = _lib.load()
    timer = launch_timer
    if timer is not None:
        ev0, ev1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev0.record()
    if is_mixed(q, k):
        ws_bytes = lib.fa4cp_attn_kv8_workspace_bytes(k.shape[0], k.shape[1], k.shape[2])
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=q.device)
        rc = lib.fa4cp_attn_fwd_kv8(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            cu_q.data_ptr(), _lib.ptr(cu_k), nseq, max_seqlen_q, q.shape[0], k.shape[0],
            q.shape[1], k.shape[1], q.shape[2], _lib.dtype_code(q.dtype), pattern,
            1 if causal else 0, float(softmax_scale), _lib.ptr(k_descale), _lib.ptr(v_descale),
            1 if accumulate else 0, ws.data_ptr(), ws.numel(), _lib.stream_of(q))
        _lib.check(rc, "attn_fwd_kv8")
        _lib.count_launches(3)
    else:
        rc = lib.fa4cp_attn_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            cu_q.data_ptr(), _lib.ptr(cu_k), nseq, max_seqlen_q, q.shape[0], k.shape[0],
            q.shape[1], k.shape[1], q.shape[2], _lib.dtype_code(q.dtype),
            _lib.dtype_code(out.dtype), pattern, 1 if causal else 0, float(softmax_scale),
            _lib.ptr(q_descale), _lib.ptr(k_descale), _lib.ptr(v_descale),
            1 if accumulate else 0, _lib.stream_of(q))
        _lib.check(rc, "attn_fwd")
        _lib.count_launches()
    if timer is not None:
        ev1.record()
        timer.append((ev0, ev1, pattern))


def b200_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool,
    softmax_scale: Optional[float] = None,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    max_seqlen_q: Optional[int] = None,
    max_seqlen_k: Optional[int] = None,
    q_descale: Optional[torch.Tensor] = None,
    k_descale: Optional[torch.Tensor] = None,
    v_descale: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Varlen attention forward; returns ``(out [T_q,H,D], lse [T_q,H] fp32 natural log)``.

    Causal masking is bottom-right aligned per sequence (key j visible to query i iff
    ``j <= i + T_k - T_q``), which is the square ``tril`` of the reference's CPU
    simulation whenever ``T_q == T_k``.  Rows that see no key get out 0, lse -inf.
    """
    _check_qkv(q, k, v)
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    dev = q.device
    t_q, t_k = q.shape[0], k.shape[0]
    if cu_seqlens_q is None:
        cu_seqlens_q = torch.tensor([0, t_q], device=dev, dtype=torch.int32)
        max_seqlen_q = t_q
    if cu_seqlens_k is None:
        cu_seqlens_k = torch.tensor([0, t_k], device=dev, dtype=torch.int32)
        max_seqlen_k = t_k
    assert max_seqlen_q is not None, "max_seqlen_q required when cu_seqlens_q is given"
    assert cu_seqlens_q.numel() == cu_seqlens_k.numel(), "cu_seqlens_q/k describe different batches"
    cu_q = cu_seqlens_q.to(device=dev, dtype=torch.int32).contiguous()
    cu_k = cu_seqlens_k.to(device=dev, dtype=torch.int32).contiguous()
    h_kv = k.shape[1]
    fp8 = q.dtype == torch.float8_e4m3fn
    kv8 = k.dtype == torch.float8_e4m3fn
    qd = norm_descale(q_descale, h_kv, dev) if fp8 else None
    kd = norm_descale(k_descale, h_kv, dev) if kv8 else None
    vd = norm_descale(v_descale, h_kv, dev) if kv8 else None
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    out = torch.empty(q.shape, dtype=out_dtype_for(q.dtype), device=dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
    nseq = cu_q.numel() - 1
    if t_q > 0 and nseq > 0:
        # rows outside every sequence of cu_seqlens_q are left unwritten (as in FA4)
        attn_into(q, k, v, out, lse, cu_q, cu_k, nseq=nseq, max_seqlen_q=int(max_seqlen_q),
                  pattern=PATTERN_VARLEN, causal=causal, softmax_scale=softmax_scale,
                  q_descale=qd, k_descale=kd, v_descale=vd, accumulate=False)
    return out, lse


# Drop-in name of the reference's per-chunk entry (fa4_ring/fa4_backend.py:58).
fa4_attn = b200_attn


def b200_attn_paged(
    q: torch.Tensor,            # [T_q, H, D]
    k_pages: torch.Tensor,      # [num_pages, page_size, H_kv, D]
    v_pages: torch.Tensor,      # [num_pages, page_size, H_kv, D]
    block_table: torch.Tensor,  # int32 [num_seqs, max_pages_per_seq]
    *,
    cu_seqlens_q: torch.Tensor,  # int32 [num_seqs + 1]
    cu_seqlens_k: torch.Tensor,  # int32 [num_seqs + 1], logical K/V lengths
    max_seqlen_q: int,
    causal: bool,
    softmax_scale: Optional[float] = None,
    q_descale: Optional[torch.Tensor] = None,
    k_descale: Optional[torch.Tensor] = None,
    v_descale: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Varlen attention over a paged K/V cache (``fa4cp_attn_fwd_paged``): the K/V rows of
    sequence j at logical position r are row ``r % page_size`` of page
    ``block_table[j, r // page_size]``.  ``page_size`` must be a multiple of 128.  Causal
    masking is bottom-right aligned per sequence, as :func:`b200_attn`.  Returns
    ``(out [T_q, H, D], lse [T_q, H] fp32 natural log)``.  Not in the reference, whose K/V is
    contiguous."""
    _lib.require_cuda(q, k_pages, v_pages, block_table)
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "pools are [pages, page, H_kv, D]"
    assert k_pages.dtype == v_pages.dtype == q.dtype, "q and the pools must share a dtype"
    num_pages, page_size, h_kv, D = k_pages.shape
    assert q.shape[2] == D and q.shape[1] % h_kv == 0
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    dev = q.device
    fp8 = q.dtype == torch.float8_e4m3fn
    qd = norm_descale(q_descale, h_kv, dev) if fp8 else None
    kd = norm_descale(k_descale, h_kv, dev) if fp8 else None
    vd = norm_descale(v_descale, h_kv, dev) if fp8 else None
    q = q.contiguous()
    bt = block_table.to(device=dev, dtype=torch.int32).contiguous()
    cu_q = cu_seqlens_q.to(device=dev, dtype=torch.int32).contiguous()
    cu_k = cu_seqlens_k.to(device=dev, dtype=torch.int32).contiguous()
    assert bt.dim() == 2 and bt.shape[0] == cu_q.numel() - 1 == cu_k.numel() - 1
    out = torch.empty(q.shape, dtype=out_dtype_for(q.dtype), device=dev)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
    lib = _lib.load()
    rc = lib.fa4cp_attn_fwd_paged(
        q.data_ptr(), k_pages.contiguous().data_ptr(), v_pages.contiguous().data_ptr(),
        bt.data_ptr(), page_size, num_pages, bt.shape[1], out.data_ptr(), lse.data_ptr(),
        cu_q.data_ptr(), cu_k.data_ptr(), cu_q.numel() - 1, int(max_seqlen_q), q.shape[0],
        q.shape[1], h_kv, D, _lib.dtype_code(q.dtype), _lib.dtype_code(out.dtype),
        1 if causal else 0, float(softmax_scale), _lib.ptr(qd), _lib.ptr(kd), _lib.ptr(vd),
        _lib.stream_of(q))
    _lib.check(rc, "attn_fwd_paged")
    _lib.count_launches()
    return out, lse


_Strides = ctypes.c_int64 * 3


@functools.lru_cache(maxsize=256)
def _strides_of(shape, stride, what: str):
    n, rows, heads, d = shape
    sp, sr, sh, sd = stride
    if sd != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    return _Strides(sp if n > 1 else rows * heads * d, sr if rows > 1 else heads * d,
                    sh if heads > 1 else d)


def pool_strides(pool: torch.Tensor, what: str):
    """(page, row, head) strides, in elements, of a pool ``[pages, page, H_kv, D]``.  Any view
    with a dense last dimension is taken as it is; the library wants the strides in multiples
    of 16 bytes.  (A pool is never copied: a copy would double the cache, and a write into it
    would be lost.)"""
    return _strides_of(pool.shape, pool.stride(), what)


def rows16(x: torch.Tensor) -> torch.Tensor:
    """``x [T, H, D]`` as rows of ``H * D`` dense elements at a 16-byte aligned token stride:
    a slice of a fused projection is taken as it is, anything else is copied (dense rows at an
    address that is not aligned, too, which ``contiguous`` would give back as they are)."""
    _, heads, d = x.shape
    token, head, elem = x.stride()
    if (elem == 1 and (head == d or heads == 1)
            and (token * x.element_size() | x.data_ptr()) & 15 == 0):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def as_i32(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """``t`` as dense int32 on ``dev``, itself if it is that.  A tensor on the host is copied, which
    waits for the stream and cannot be captured into a graph."""
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    return t.to(device=dev, dtype=torch.int32).contiguous()


@functools.lru_cache(maxsize=64)
def _tree_workspace_bytes(heads: int, heads_kv: int, dim: int, max_seqlen_q: int) -> int:
    return max(_lib.load().fa4cp_attn_paged_tree_workspace_bytes(heads, heads_kv, dim, max_seqlen_q), 16)


def b200_attn_paged_tree(
    q: torch.Tensor,            # [T, H, D]
    k_pages: torch.Tensor,      # [num_pages, page_size, H_kv, D]
    v_pages: torch.Tensor,      # [num_pages, page_size, H_kv, D]
    block_table: torch.Tensor,  # int32 [num_seqs, max_pages_per_seq]
    *,
    cu_seqlens_q: torch.Tensor,  # int32 [num_seqs + 1]
    seq_lens: torch.Tensor,      # int32 [num_seqs], cached tokens, the step's own included
    max_seqlen_q: int,
    tree_mask: Optional[torch.Tensor] = None,  # int64 [T, words]
    softmax_scale: Optional[float] = None,
    q_descale: Optional[torch.Tensor] = None,
    k_descale: Optional[torch.Tensor] = None,
    v_descale: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of a few new tokens a request over its paged K/V cache
    (``fa4cp_attn_fwd_paged_tree``): decode steps and the verification of drafted trees.

    Request ``j`` brings the tokens ``cu_seqlens_q[j] .. cu_seqlens_q[j + 1]``; their K/V are
    the last rows of its ``seq_lens[j]`` cached tokens (see
    :mod:`fa4_ring.paged_cache`).  Every token sees all rows before them, and of the new rows
    those that its ``tree_mask`` bits name (:func:`fa4_ring.paged_tree_mask`): bit ``m`` of
    word ``w`` is node ``64 w + m`` of its request.  Without a mask a token sees the new rows
    up to its own (bottom-right causal, as :func:`b200_attn`); one token a request is decode.

    q is f16 / bf16 with K/V of its dtype, or bf16 / e4m3 with e4m3 K/V (and their descales,
    scalar, ``[H_kv]`` or ``(1, H_kv)``; an f16 q over e4m3 K/V, which has more bits than the two
    e4m3 terms that a bf16 q is split into, is refused); head_dim 64, 128 or 256; page_size 16, 32,
    64 or a multiple of 128; ``max_seqlen_q`` bounds the requests' new tokens.  The pools may be
    views of another layout.  Long caches are split over the GPU whatever the batch.  The weights
    are rounded to the 16-bit type of the V that they multiply (f16 for e4m3 V), sums and
    statistics are in fp32; scores are below 2^26 in log2 units.  Returns ``(out [T, H, D], lse [T, H] fp32 natural log)``;
    out has q's dtype (bf16 for e4m3).  A row that sees no key gets out 0, lse -inf.  What lies
    behind ``seq_lens`` in a page never reaches the result, nor does what a token does not see.
    Rows outside ``cu_seqlens_q`` are left unwritten.  ``cu_seqlens_q``, ``seq_lens`` or descales of
    several heads that are on the host are copied to q's device, which waits for the stream and
    cannot be captured into a graph."""
    _lib.require_cuda(q, k_pages, v_pages, block_table, tree_mask)
    assert q.dim() == 3, "expected a [T, H, D] q"
    assert k_pages.dim() == 4 and k_pages.shape == v_pages.shape, "pools are [pages, page, H_kv, D]"
    assert k_pages.dtype == v_pages.dtype, "the pools must share a dtype"
    num_pages, page_size, h_kv, D = k_pages.shape
    T, H, dq = q.shape
    assert dq == D and H % h_kv == 0, f"q [{T}, {H}, {dq}] does not fit H_kv={h_kv}, D={D}"
    dev = q.device
    assert k_pages.device == v_pages.device == dev, "q and the pools must be on one device"
    nseq = cu_seqlens_q.numel() - 1
    assert block_table.dim() == 2 and block_table.shape[0] == nseq == seq_lens.numel(), (
        "block_table, cu_seqlens_q and seq_lens describe different batches")
    words = 0
    if tree_mask is not None:
        assert tree_mask.dim() == 2 and tree_mask.shape[0] == T and tree_mask.dtype == torch.int64, (
            "tree_mask is int64 [T, words]")
        assert tree_mask.device == dev, "tree_mask must be on q's device"
        words = tree_mask.shape[1]
        tree_mask = tree_mask.contiguous()
    qd, kd = norm_descale(q_descale, h_kv, dev), norm_descale(k_descale, h_kv, dev)
    vd = norm_descale(v_descale, h_kv, dev)
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    q = rows16(q)
    ks, vs = pool_strides(k_pages, "k_pages"), pool_strides(v_pages, "v_pages")
    bt, cu, lens = as_i32(block_table, dev), as_i32(cu_seqlens_q, dev), as_i32(seq_lens, dev)
    out = q.new_empty((T, H, D), dtype=out_dtype_for(q.dtype))
    lse = q.new_empty((T, H), dtype=torch.float32)
    lib = _lib.load()
    with _lib.on_device(dev):
        ws = q.new_empty(_tree_workspace_bytes(H, h_kv, D, max_seqlen_q), dtype=torch.uint8)
        rc = lib.fa4cp_attn_fwd_paged_tree(
            q.data_ptr(), q.stride(0), k_pages.data_ptr(), v_pages.data_ptr(), ks, vs,
            bt.data_ptr(), page_size, num_pages, bt.shape[1], out.data_ptr(), lse.data_ptr(),
            cu.data_ptr(), lens.data_ptr(), nseq, int(max_seqlen_q), T, H, h_kv, D,
            _lib.dtype_code(q.dtype), _lib.dtype_code(k_pages.dtype), _lib.ptr(tree_mask), words,
            float(softmax_scale), _lib.ptr(qd), _lib.ptr(kd), _lib.ptr(vd), ws.data_ptr(),
            ws.numel(), _lib.stream_of(q))
    _lib.check(rc, "attn_fwd_paged_tree")
    _lib.count_launches(2)  # the attention, and the join of its parts
    return out, lse
