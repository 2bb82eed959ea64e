"""Refusals of the paged-cache entry points, before any CUDA call (no GPU needed)."""

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from fa4_ring import _build, _lib
    _build.build()
    return _lib.load()


P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(264)
S = (ctypes.c_int64 * 3)(16 * 2 * 128, 2 * 128, 128)


def _tree(lib, **kw):
    a = dict(q=P, qs=1024, k=P, v=P, ks=S, vs=S, bt=P, page=16, pages=4, maxp=4, out=P, lse=P, cu=P,
             lens=P, nseq=1, maxq=4, T=4, H=8, hk=2, D=128, qd=1, kd=1, mask=None, words=0, scale=0.1,
             qds=None, kds=None, vds=None, ws=P, wsb=1 << 40)
    a.update(kw)
    rc = lib.fa4cp_attn_fwd_paged_tree(*a.values(), None)
    return rc, lib.fa4cp_last_error()


@pytest.mark.parametrize("kw,rc,needle", [
    (dict(H=7), -1, b"multiple"),
    (dict(hk=0), -1, b"multiple"),
    (dict(page=8), -1, b"page_size"),
    (dict(page=48), -1, b"page_size"),
    (dict(page=192), -1, b"page_size"),
    (dict(page=0), -1, b"page_size"),
    (dict(D=96), -2, b"head_dim"),
    (dict(qd=2), -1, b"dtype"),
    (dict(qd=3, kd=1), -1, b"dtype"),
    (dict(qd=0, kd=1), -1, b"dtype"),
    (dict(kds=P), -1, b"descale"),
    (dict(qds=P), -1, b"descale"),
    (dict(scale=0.0), -1, b"softmax_scale"),
    (dict(scale=float("nan")), -1, b"softmax_scale"),
    (dict(mask=P, words=0), -1, b"mask_words"),
    (dict(nseq=0), -1, b"request"),
    (dict(cu=None), -1, b"request"),
    (dict(T=-1), -1, b"sizes"),
    (dict(maxp=0), -1, b"sizes"),
    (dict(q=ODD), -1, b"aligned"),
    (dict(qs=1025), -1, b"aligned"),
    (dict(ks=(ctypes.c_int64 * 3)(4096, 257, 128)), -1, b"16 bytes"),
    (dict(vs=(ctypes.c_int64 * 3)(4096, 256, -128)), -1, b"16 bytes"),
    (dict(out=None), -1, b"null"),
    (dict(bt=None), -1, b"null"),
])
def test_attention_refuses(lib, kw, rc, needle):
    got, text = _tree(lib, **kw)
    assert got == rc and needle in text, text


def test_attention_of_nothing(lib):
    assert _tree(lib, T=0)[0] == 0 and _tree(lib, maxq=0)[0] == 0
    assert lib.fa4cp_attn_paged_tree_workspace_bytes(8, 2, 128, 4) >= 0
    assert lib.fa4cp_attn_paged_tree_workspace_bytes(8, 0, 128, 4) == -1


def test_block_tables_refuse(lib):
    def plan(nseq=1, free=P, nfree=4, page=16, maxp=4, tin=None, tout=P, slots=P, n=4, cached=P):
        return lib.fa4cp_paged_block_tables(cached, P, nseq, free, nfree, None, page, maxp, tin, tout,
                                            slots, n, P, P, P, P, None), lib.fa4cp_last_error()
    for kw, needle in ((dict(nseq=0), b"nseq"), (dict(page=0), b"page_size"), (dict(maxp=0), b"sizes"),
                       (dict(nfree=-1), b"sizes"), (dict(n=-1), b"sizes"), (dict(free=None), b"null"),
                       (dict(slots=None), b"null"), (dict(cached=None), b"null"), (dict(tin=P), b"old one")):
        rc, text = plan(**kw)
        assert rc == -1 and needle in text, (kw, text)


def test_tree_mask_refuses(lib):
    def mask(parents=P, cu=P, nseq=1, total=4, nodes=4, out=P):
        return lib.fa4cp_paged_tree_mask(parents, cu, nseq, total, nodes, out, None), lib.fa4cp_last_error()
    for kw, needle in ((dict(nodes=0), b"max_nodes"), (dict(nodes=4097), b"max_nodes"), (dict(nseq=0), b"request"),
                       (dict(cu=None), b"request"), (dict(total=-1), b"sizes"), (dict(out=None), b"null")):
        rc, text = mask(**kw)
        assert rc == -1 and needle in text, (kw, text)
    assert mask(total=0)[0] == 0


def test_write_refuses(lib):
    def write(k=P, kst=256, kp=P, ks=S, vs=S, pages=4, page=16, slots=P, n=4, hk=2, D=128, src=1, dst=1, kds=None):
        return lib.fa4cp_paged_kv_write(k, P, kst, 256, kp, P, ks, vs, pages, page, slots, n, hk, D, src, dst,
                                        kds, None, None), lib.fa4cp_last_error()
    for kw, needle in ((dict(src=0), b"dtype"), (dict(src=3), b"dtype"), (dict(src=2, dst=3), b"dtype"),
                       (dict(src=2, dst=2), b"dtype"), (dict(dst=9), b"dtype"), (dict(kds=P), b"descales"),
                       (dict(D=12), b"16 bytes"), (dict(dst=3, D=24), b"16 bytes"), (dict(hk=0), b"sizes"),
                       (dict(page=0), b"sizes"), (dict(n=-1), b"sizes"), (dict(k=ODD), b"aligned"),
                       (dict(kst=260), b"aligned"), (dict(kp=ODD), b"aligned"), (dict(kp=None), b"null"),
                       (dict(slots=None), b"null"), (dict(ks=(ctypes.c_int64 * 3)(4096, 4, 128)), b"aligned")):
        rc, text = write(**kw)
        assert rc == -1 and needle in text, (kw, text)
    assert write(n=0)[0] == 0 and write(pages=0)[0] == 0


def test_accept_refuses(lib):
    def accept(kp=P, ks=S, pages=4, page=16, maxp=4, nseq=1, acc=P, A=4, hk=2, D=128, dt=1, lens=P):
        return lib.fa4cp_paged_kv_accept(kp, P, ks, S, pages, page, P, maxp, P, P, nseq, acc, A, hk, D, dt, lens,
                                         None), lib.fa4cp_last_error()
    for kw, needle in ((dict(A=1025), b"max_accept"), (dict(A=-1), b"max_accept"), (dict(nseq=0), b"nseq"),
                       (dict(dt=2), b"dtype"), (dict(D=4), b"16 bytes"), (dict(page=0), b"sizes"),
                       (dict(maxp=0), b"sizes"), (dict(acc=None), b"null"), (dict(kp=ODD), b"aligned"),
                       (dict(lens=None), b"null")):
        rc, text = accept(**kw)
        assert rc == -1 and needle in text, (kw, text)
