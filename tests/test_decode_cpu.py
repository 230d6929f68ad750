"""CPU tests of the token-generation operators' boundary: argument checks that
come before any device work, fake kernels' shapes, the rotary tables."""
import ctypes
import math

import pytest
import torch

import cuda_transformer_b200 as cb

P = ctypes.c_void_p(256)
S3 = (ctypes.c_int64 * 3)(64, 64, 1)
S4 = (ctypes.c_int64 * 4)(1024, 512, 64, 1)


def attention(**kw):
    a = dict(q=P, qs=S3, k=P, ks=S4, v=P, vs=S4, table=P, ts=2, lens=P, out=P, lse=None, batch=3,
             heads=4, kv=2, dim=64, pages=4, page=8, width=2, scale=0.125, act=cb.DTYPE_F32,
             cache=cb.DTYPE_F32, ws=P, wsb=1 << 26, stream=None)
    a.update(kw)
    return cb.lib().ct_paged_attention(*a.values())


def append(**kw):
    a = dict(q=P, qs=S3, k=P, ks=S3, v=P, vs=S3, qo=P, ko=None, cos=P, sin=P, kc=P, kcs=S4, vc=P,
             vcs=S4, table=P, ts=2, ids=None, pos=P, tokens=3, heads=4, kv=2, dim=64, rot=64,
             inter=0, maxpos=16, batch=3, pages=4, page=8, width=2, act=cb.DTYPE_F32,
             cache=cb.DTYPE_F32, stream=None)
    a.update(kw)
    return cb.lib().ct_kv_append(*a.values())


def logits(**kw):
    a = dict(x=P, ld=100, dtype=cb.DTYPE_F32, out=ctypes.c_void_p(4096), old=100, rows=2,
             vocab=100, tokens=P, tld=5, width=5, lens=None, plens=None, rep=None, freq=None,
             pres=None, ids=None, ild=0, values=None, vld=0, n=0, mask=None, mld=0, stream=None)
    a.update(kw)
    return cb.lib().ct_logits_process(*a.values())


def test_attention_refusals():
    bad, dim, layout = (cb.CT_ERR_INVALID_ARGUMENT, cb.CT_ERR_UNSUPPORTED_HEAD_DIM,
                        cb.CT_ERR_UNSUPPORTED_LAYOUT)
    odd = (ctypes.c_int64 * 4)(1024, 512, 66, 1)
    wide = (ctypes.c_int64 * 4)(1024, 512, 64, 2)
    minus = (ctypes.c_int64 * 4)(1024, 512, -64, 1)
    for want, kw in ((bad, dict(batch=-1)), (bad, dict(heads=3)), (bad, dict(kv=0)),
                     (bad, dict(page=0)), (bad, dict(pages=-1)), (bad, dict(width=2 ** 31)),
                     (bad, dict(width=2 ** 20, page=2 ** 11)), (bad, dict(batch=2 ** 30)),
                     (bad, dict(act=cb.DTYPE_BF16)), (bad, dict(act=3, cache=3)),
                     (bad, dict(act=cb.DTYPE_BF16, cache=cb.DTYPE_F16)), (dim, dict(dim=48)),
                     (bad, dict(q=None)), (bad, dict(lens=None)), (bad, dict(out=None)),
                     (bad, dict(table=None)), (bad, dict(k=None)), (layout, dict(ks=odd)),
                     (layout, dict(vs=wide)), (layout, dict(ks=minus)),
                     (layout, dict(v=ctypes.c_void_p(260))), (bad, dict(out=ctypes.c_void_p(260))),
                     (cb.CT_OK, dict(batch=0)), (cb.CT_OK, dict(heads=0))):
        assert attention(**kw) == want, kw


def test_append_refusals():
    bad, layout = cb.CT_ERR_INVALID_ARGUMENT, cb.CT_ERR_UNSUPPORTED_LAYOUT
    wide = (ctypes.c_int64 * 3)(64, 64, 2)
    for want, kw in ((bad, dict(tokens=-1)), (bad, dict(rot=7)), (bad, dict(rot=66)),
                     (bad, dict(cos=None)), (bad, dict(maxpos=-1)), (bad, dict(q=None)),
                     (bad, dict(qo=None)), (bad, dict(k=None)), (bad, dict(pos=None)),
                     (bad, dict(kc=None)), (bad, dict(table=None)), (bad, dict(act=cb.DTYPE_F16)),
                     (cb.CT_ERR_UNSUPPORTED_HEAD_DIM, dict(dim=80)), (layout, dict(ks=wide)),
                     (layout, dict(qs=wide)), (cb.CT_OK, dict(tokens=0))):
        assert append(**kw) == want, kw


def test_logits_refusals():
    bad = cb.CT_ERR_INVALID_ARGUMENT
    for want, kw in ((bad, dict(rows=-1)), (bad, dict(vocab=0)), (bad, dict(ld=99)),
                     (bad, dict(old=99)), (bad, dict(dtype=5)), (bad, dict(width=-1)),
                     (bad, dict(n=3)), (bad, dict(n=-1)), (bad, dict(x=None)), (bad, dict(out=None)),
                     (bad, dict(out=P, dtype=cb.DTYPE_BF16)), (bad, dict(out=P, old=128)),
                     (bad, dict(mask=P, mld=-1)), (cb.CT_OK, dict(rows=0))):
        assert logits(**kw) == want, kw


def test_workspace_query():
    lib = cb.lib()
    assert lib.ct_paged_attention_workspace_size(8, 0, 64) == 0
    assert lib.ct_paged_attention_workspace_size(-1, 2, 64) == 0
    assert 0 <= lib.ct_paged_attention_workspace_size(64, 1, 128) < 1 << 25


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from cuda_transformer import ops
    with FakeTensorMode():
        k = torch.empty(4, 2, 8, 64, dtype=torch.bfloat16)
        table, n = torch.empty(3, 2, dtype=torch.int32), torch.empty(3, dtype=torch.int32)
        q = torch.empty(3, 4, 64)
        out, lse = ops.paged_attention(q, k, k, table, n)
        assert out.shape == q.shape and lse.shape == (3, 4) and lse.dtype == torch.float32
        kn = torch.empty(3, 2, 64)
        q_out, k_out = ops.kv_append_(k, k, kn, kn, table, n, q=q)
        assert q_out.shape == q.shape and k_out.numel() == 0
        q_out, k_out = ops.kv_append_(k, k, kn, kn, table, n, want_k=True)
        assert q_out.numel() == 0 and k_out.shape == kn.shape
        x = torch.empty(3, 50, dtype=torch.float16)
        y = ops.logits_process(x)
        assert y.shape == x.shape and y.dtype == torch.float32


def test_cpu_tensors_are_refused():
    from cuda_transformer import ops
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.logits_process(torch.zeros(2, 5))


def test_rotary_tables():
    from cuda_transformer import ops
    cos, sin = ops.rotary_tables(100001, 8)
    assert cos.shape == sin.shape == (100001, 4) and cos.dtype == torch.float32
    for p, i in ((0, 3), (1, 0), (100000, 0), (100000, 2)):
        angle = p * 10000.0 ** (-2 * i / 8)
        assert abs(cos[p, i].item() - math.cos(angle)) < 1e-7
        assert abs(sin[p, i].item() - math.sin(angle)) < 1e-7


def test_page_pool():
    from cuda_transformer_b200.generate_case import PagePool

    pool = PagePool(6, 4, 2, 4, "cpu")
    pool.reserve(0, 9)
    pool.reserve(0, 5)   # fewer than it has: nothing changes
    pool.reserve(1, 1)
    assert [len(p) for p in pool.owned] == [3, 1] and len(pool.free) == 2
    assert pool.table[0, :3].tolist() == pool.owned[0] and len(set(sum(pool.owned, []))) == 4
    pool.reserve(0, 16)
    with pytest.raises(RuntimeError):
        pool.reserve(1, 16)
    with pytest.raises(ValueError):
        pool.reserve(1, 17)
    pool.release(0)
    pool.reserve(1, 16)
    assert len(pool.free) == 2 and pool.table[1].tolist() == pool.owned[1]


def test_attention_size_bound():
    """Shares are products of the tiles of all items and the CTAs, in 64 bits: sizes whose
    products could pass them are refused before any device call."""
    bad = cb.CT_ERR_INVALID_ARGUMENT
    big = dict(heads=1 << 10, kv=1, width=1 << 20, page=1 << 9)      # 2^26 tiles of 8 keys
    assert attention(batch=1 << 20, **big) == bad                    # 2^30 heads
    assert attention(batch=1 << 17, **big) == bad
    for ok in (dict(big, batch=1 << 15), dict(batch=(1 << 20) - 1, heads=1 << 11, kv=1, width=1,
                                              page=128)):
        # (accepted up to the workspace)
        assert attention(wsb=0, **ok) == cb.CT_ERR_WORKSPACE_TOO_SMALL


def test_rotary_tables_of_an_odd_part_are_refused():
    from cuda_transformer import ops
    for rot in (7, -2):
        with pytest.raises(RuntimeError):
            ops.rotary_tables(4, rot)


def test_strides_of_single_elements_do_not_matter():
    """A dimension of one element may have any stride (imported tensors have 1 there), also
    where others must be multiples of 16 bytes or not negative; a table without rows has no
    address.  (Accepted up to the workspace, or the device.)"""
    odd = (ctypes.c_int64 * 4)(1, -3, 64, 1)
    assert attention(ks=odd, vs=odd, pages=1, kv=1, wsb=0) == cb.CT_ERR_WORKSPACE_TOO_SMALL
    one = (ctypes.c_int64 * 4)(128, 64, 7, 1)
    assert attention(ks=one, vs=one, page=1, wsb=0) == cb.CT_ERR_WORKSPACE_TOO_SMALL
    assert attention(ks=one, vs=one, wsb=0) == cb.CT_ERR_UNSUPPORTED_LAYOUT
    refused = (cb.CT_ERR_INVALID_ARGUMENT, cb.CT_ERR_UNSUPPORTED_LAYOUT)
    assert attention(ks=odd, vs=odd, pages=1, kv=2, wsb=0) in refused
    if not torch.cuda.is_available():   # (the addresses are made up)
        assert append(kcs=odd, vcs=odd, pages=1, kv=1) not in refused
        assert append(batch=0, table=None) not in refused
