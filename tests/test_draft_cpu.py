"""CPU tests of the speculative-decoding operators' boundary: argument checks
that come before any device work, fake kernels' shapes."""
import ctypes

import pytest
import torch

import cuda_transformer_b200 as cb

P = ctypes.c_void_p(256)
S2 = (ctypes.c_int64 * 2)(400, 100)
S4 = (ctypes.c_int64 * 4)(1024, 512, 64, 1)
BAD, DIM, LAYOUT = (cb.CT_ERR_INVALID_ARGUMENT, cb.CT_ERR_UNSUPPORTED_HEAD_DIM,
                    cb.CT_ERR_UNSUPPORTED_LAYOUT)


def attention(**kw):
    a = dict(q=P, qs=S4, k=P, ks=S4, v=P, vs=S4, table=P, ts=2, context=P, lens=None, mask=None,
             ms=None, out=P, lse=None, batch=3, drafts=5, heads=4, kv=2, dim=64, pages=4, page=8,
             width=2, scale=0.125, act=cb.DTYPE_F32, cache=cb.DTYPE_F32, ws=P, wsb=1 << 30,
             stream=None)
    a.update(kw)
    return cb.lib().ct_tree_attention(*a.values())


def verify(**kw):
    a = dict(target=P, ts=S2, draft=P, ds=S2, dtype=cb.DTYPE_F32, tokens=P, tld=4, parents=P, pld=4,
             lens=None, uniform=P, uld=4, new=P, path=P, counts=P, batch=3, drafts=4, vocab=100,
             stream=None)
    a.update(kw)
    return cb.lib().ct_verify_drafts(*a.values())


def pointers(n, first=256):
    return (ctypes.c_void_p * n)(*[first] * n)


def strides(n, one=(1024, 512, 64, 1)):
    return (ctypes.c_int64 * (4 * n))(*list(one) * n)


def compact(**kw):
    a = dict(caches=pointers(2), strides=strides(2), n=2, table=P, ts=2, context=P, keep=P, kld=4,
             counts=P, batch=3, drafts=4, kv=2, dim=64, pages=4, page=8, width=2,
             dtype=cb.DTYPE_F32, stream=None)
    a.update(kw)
    return cb.lib().ct_kv_compact(*a.values())


def copy(**kw):
    a = dict(caches=pointers(2), strides=strides(2), n=2, src=P, dst=P, count=3, kv=2, dim=64,
             pages=4, page=8, dtype=cb.DTYPE_F32, stream=None)
    a.update(kw)
    return cb.lib().ct_kv_copy_pages(*a.values())


def test_attention_refusals():
    odd = (ctypes.c_int64 * 4)(1024, 512, 66, 1)
    wide = (ctypes.c_int64 * 4)(1024, 512, 64, 2)
    minus = (ctypes.c_int64 * 4)(1024, 512, -64, 1)
    most = cb.CT_TREE_ATTENTION_MAX_DRAFTS
    for want, kw in ((BAD, dict(batch=-1)), (BAD, dict(heads=3)), (BAD, dict(kv=0)),
                     (BAD, dict(drafts=-1)), (BAD, dict(drafts=most + 1)), (BAD, dict(page=0)),
                     (BAD, dict(pages=-1)), (BAD, dict(width=2 ** 31)),
                     (BAD, dict(width=2 ** 20, page=2 ** 11)), (BAD, dict(batch=2 ** 30)),
                     (BAD, dict(batch=2 ** 20, drafts=2 ** 10)),
                     (BAD, dict(batch=2 ** 20, drafts=2 ** 8, width=2 ** 20, page=2 ** 9)),
                     (BAD, dict(heads=2 ** 18)), (BAD, dict(act=cb.DTYPE_BF16)),
                     (BAD, dict(act=3, cache=3)),
                     (BAD, dict(act=cb.DTYPE_BF16, cache=cb.DTYPE_F16)), (DIM, dict(dim=48)),
                     (BAD, dict(q=None)), (BAD, dict(qs=None)), (BAD, dict(context=None)),
                     (BAD, dict(out=None)), (BAD, dict(mask=P)), (BAD, dict(table=None)),
                     (BAD, dict(k=None)), (LAYOUT, dict(ks=odd)), (LAYOUT, dict(vs=wide)),
                     (LAYOUT, dict(ks=minus)), (LAYOUT, dict(v=ctypes.c_void_p(260))),
                     (BAD, dict(out=ctypes.c_void_p(260))), (cb.CT_OK, dict(batch=0)),
                     (cb.CT_OK, dict(heads=0)), (cb.CT_OK, dict(drafts=0))):
        assert attention(**kw) == want, kw


def test_attention_workspace():
    size = cb.lib().ct_tree_attention_workspace_size
    for bad in ((-1, 4, 2, 64), (4, -1, 2, 64), (4, 4, 0, 64), (4, 5, 2, 64), (4, 4, 2, 0)):
        assert size(*bad) == 0
    need = size(5, 4, 2, 64)
    assert 0 <= size(16384, 64, 1, 128) < 1 << 28
    if need > 0:
        assert attention(wsb=need - 1) == cb.CT_ERR_WORKSPACE_TOO_SMALL
        assert attention(ws=None, wsb=need) == cb.CT_ERR_WORKSPACE_TOO_SMALL
        assert attention(ws=ctypes.c_void_p(264)) == BAD


def test_verify_refusals():
    minus = (ctypes.c_int64 * 2)(-400, 100)
    for want, kw in ((BAD, dict(batch=-1)), (BAD, dict(drafts=0)),
                     (BAD, dict(drafts=cb.CT_VERIFY_DRAFTS_MAX + 1)), (BAD, dict(vocab=0)),
                     (BAD, dict(vocab=2 ** 30)), (BAD, dict(dtype=3)), (BAD, dict(tld=-1)),
                     (BAD, dict(pld=-1)), (BAD, dict(uld=-1)), (BAD, dict(uniform=None)),
                     (BAD, dict(ds=None)), (BAD, dict(target=None)), (BAD, dict(ts=None)),
                     (BAD, dict(tokens=None)), (BAD, dict(new=None)), (BAD, dict(path=None)),
                     (BAD, dict(counts=None)), (LAYOUT, dict(ts=minus)), (LAYOUT, dict(ds=minus)),
                     (cb.CT_OK, dict(batch=0))):
        assert verify(**kw) == want, kw


def test_move_refusals():
    for want, kw in ((BAD, dict(n=-1)), (BAD, dict(kv=0)), (BAD, dict(kv=2 ** 17)),
                     (BAD, dict(dim=0)), (BAD, dict(dim=2 ** 17)), (BAD, dict(pages=-1)),
                     (BAD, dict(page=0)), (BAD, dict(page=2 ** 30)), (BAD, dict(dtype=3)),
                     (BAD, dict(caches=None)), (BAD, dict(strides=None)),
                     (BAD, dict(caches=pointers(2, None))),
                     (LAYOUT, dict(strides=strides(2, (1024, 512, 64, 2)))),
                     (LAYOUT, dict(strides=strides(2, (1024, -512, 64, 1)))),
                     (cb.CT_OK, dict(n=0)), (cb.CT_OK, dict(pages=0))):
        assert compact(**kw) == want, kw
        assert copy(**kw) == want, kw
    for want, kw in ((BAD, dict(batch=-1)), (BAD, dict(drafts=-1)), (BAD, dict(width=-1)),
                     (BAD, dict(width=2 ** 28)), (BAD, dict(kld=-1)), (BAD, dict(table=None)),
                     (BAD, dict(context=None)), (BAD, dict(keep=None)), (BAD, dict(counts=None)),
                     (cb.CT_OK, dict(batch=0)), (cb.CT_OK, dict(drafts=0))):
        assert compact(**kw) == want, kw
    for want, kw in ((BAD, dict(count=-1)), (BAD, dict(src=None)), (BAD, dict(dst=None)),
                     (cb.CT_OK, dict(count=0))):
        assert copy(**kw) == want, kw


def test_one_cache_twice_is_refused():
    """Moving it up twice at once would lose tokens."""
    one = (ctypes.c_void_p * 3)(256, 512, 256)
    assert compact(caches=one, strides=strides(3), n=3) == BAD
    assert compact(caches=one, strides=strides(3), n=3, pages=0) == cb.CT_OK


def test_strides_of_single_elements_are_not_looked_at():
    """A head dim of one element has any stride."""
    one = dict(dim=1, pages=0, strides=strides(2, (64, 32, 8, 7)))
    assert compact(**one) == copy(**one) == cb.CT_OK
    two = dict(one, dim=2)
    assert compact(**two) == copy(**two) == LAYOUT


def test_append_refusals_with_angles():
    """ct_kv_append_ex checks what ct_kv_append checks."""
    S3 = (ctypes.c_int64 * 3)(64, 64, 1)
    a = dict(q=P, qs=S3, k=P, ks=S3, v=P, vs=S3, qo=P, ko=None, cos=P, sin=P, kc=P, kcs=S4, vc=P,
             vcs=S4, table=P, ts=2, ids=None, pos=P, angles=P, tokens=3, heads=4, kv=2, dim=64,
             rot=64, inter=0, maxpos=16, batch=3, pages=4, page=8, width=2, act=cb.DTYPE_F32,
             cache=cb.DTYPE_F32, stream=None)
    for want, kw in ((BAD, dict(tokens=-1)), (BAD, dict(rot=7)), (BAD, dict(pos=None)),
                     (DIM, dict(dim=80)), (cb.CT_OK, dict(tokens=0))):
        assert cb.lib().ct_kv_append_ex(*{**a, **kw}.values()) == want, kw


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from cuda_transformer import ops
    with FakeTensorMode():
        k = torch.empty(4, 2, 8, 64, dtype=torch.bfloat16)
        table, n = torch.empty(3, 2, dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        q = torch.empty(3, 5, 4, 64)
        out, lse = ops.tree_attention(q, k, k, table, n)
        assert out.shape == q.shape and lse.shape == (3, 5, 4) and lse.dtype == torch.float32
        tokens = torch.empty(3, 5, dtype=torch.int64)
        new, path, counts = ops.verify_drafts(torch.empty(3, 5, 100), tokens)
        assert new.shape == path.shape == (3, 5) and counts.shape == (3,)
        assert (new.dtype, path.dtype, counts.dtype) == (torch.int64, torch.int32, torch.int32)
        assert ops.kv_compact_([k, k], table, n, path, counts) is None
        assert ops.kv_copy_pages_([k, k], n, n) is None
        kn = torch.empty(3, 2, 64)
        ops.kv_append_(k, k, kn, kn, table, n, rotary_positions=n)


def test_cpu_tensors_are_refused():
    from cuda_transformer import ops
    ids = torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ops.verify_drafts(torch.zeros(2, 3, 5), ids),
                 lambda: ops.kv_copy_pages_([torch.zeros(2, 1, 4, 8)], ids[0].int(), ids[1].int())):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
