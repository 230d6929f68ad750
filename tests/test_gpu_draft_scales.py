"""tree_attention with activations and scales of any magnitude: the scores are what
counts, not how they are divided between q and the scale."""
import pytest
import torch

from .test_gpu_decode import BF16, F16, F32, gen, make_cache
from .test_gpu_draft import check, ints, ops, pack, tree_bits  # noqa: F401
from .test_gpu_draft_rounding import norm_check

pytestmark = pytest.mark.gpu

CONTEXTS = [300, 0, 1500]


def case(n, heads, kv, dim, page, cache, seed):
    g = gen(seed)
    k, v, table = make_cache([c + n for c in CONTEXTS], kv, dim, page, cache, "head", g)
    q = torch.randn(3, n, heads, dim, generator=g, device="cuda")
    return q, k, v, table, tree_bits(3, n, seed)


@pytest.mark.parametrize("cache", [F32, BF16, F16])
@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e-3, 1e5, 1e30])
@pytest.mark.parametrize("n,heads,kv,dim", [(2, 6, 6, 64), (5, 6, 2, 128), (9, 6, 2, 32),
                                            (24, 8, 2, 64)])
def test_fp32_queries_of_any_size(cuda_device, ops, cache, size, n, heads, kv, dim):  # noqa: F811
    """Scores of the order of 1 from small and from large queries; some heads of the
    thousandth part, whose rows have factors of their own."""
    q, k, v, table, bits = case(n, heads, kv, dim, 16, cache, n)
    q[:, :, ::3] *= 1e-3
    q *= size
    scale = dim ** -0.5 / size
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits), scale=scale)
    norm_check(q, k, v, table, CONTEXTS, [n] * 3, bits, 16, out, scale)
    check(q, k, v, table, CONTEXTS, [n] * 3, bits, 16, (out, lse), scale)


def test_an_infinite_query_is_its_rows_alone(cuda_device, ops):  # noqa: F811
    """q of 1e5 beside it is still finite in f16's terms."""
    q, k, v, table, bits = case(5, 4, 2, 64, 16, F16, 3)
    q *= 1e5
    want = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits), scale=1e-6)[0]
    q[1, 2, 1, 7] = torch.inf
    out, _ = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits), scale=1e-6)
    assert out[1, 2, 1].isnan().all()
    out[1, 2, 1] = want[1, 2, 1]
    assert torch.equal(out, want) and want.isfinite().all()


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("n,heads,kv,dim,page", [(24, 8, 2, 64, 16), (9, 6, 2, 128, 24),
                                                 (40, 5, 1, 128, 8), (33, 16, 2, 64, 64),
                                                 (4, 6, 2, 64, 16), (30, 4, 4, 64, 5)])
def test_scales_of_16_bit_activations(cuda_device, ops, kind, n, heads, kv, dim, page):  # noqa: F811
    """A negative, a zero and a large scale (scores of hundreds, one key far above the
    rest, late and early), a query that is read element by element: on tcgen05 and on
    the warps' products."""
    q, k, v, table, bits = case(n, heads, kv, dim, page, kind, n + dim)
    for b, j in ((0, 290), (2, 3)):
        k[int(table[b, j // page]), :, j % page] = 3 * q[b, 2, ::heads // kv].to(kind)
    q, mask = q.to(kind), pack(bits)
    args = (k, v, table, ints(CONTEXTS), None, mask)
    for scale in (dim ** -0.5, 1.0, -0.3, 0.0, 4.0):
        got = ops.tree_attention(q, *args, scale)
        check(q, k, v, table, CONTEXTS, [n] * 3, bits, page, got, scale)
        if scale < 0:  # only q's sign turns
            other = ops.tree_attention(-q, *args, -scale)
            assert all(torch.equal(a, b) for a, b in zip(got, other))
        if scale in (dim ** -0.5, 0.0):
            norm_check(q, k, v, table, CONTEXTS, [n] * 3, bits, page, got[0], scale)
        turned = q.transpose(2, 3).contiguous().transpose(2, 3)
        shifted = torch.nn.functional.pad(q, (3, 0))[..., 3:]
        for view in (turned, shifted):
            again = ops.tree_attention(view, *args, scale)
            assert all(torch.equal(a, b) for a, b in zip(got, again))
