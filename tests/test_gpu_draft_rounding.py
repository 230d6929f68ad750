"""How exact tree_attention is: errors against 64 bits by their norm, which shows the
loss of a term that bounds for single elements would admit."""
import pytest
import torch

from .test_gpu_decode import BF16, F16, F32, TYPES, gen, make_cache
from .test_gpu_draft import ints, ops, pack, reference, tree_bits  # noqa: F401

pytestmark = pytest.mark.gpu

CONTEXTS = [300, 40, 2000]


def norm_check(q, k, v, table, context, drafts, bits, page, out, scale):
    """Tolerance, all of it relative to the norm of O.  Arithmetic: terms of q, k, the
    weights and v that keep 22 bits, FP32 scores and sums, the tensor core's cut-off sums:
    each 2^-22 at most of values of the order of 1 (inputs are unit normal, so are the
    scores), six of them below 2^-19.  16-bit results are rounded once: as far as the
    64-bit results are when they are rounded (5 % for other neighbours of a border).
    16-bit activations have weights of two terms: 2^-17 (bf16), 2^-21 (f16) of sum w|v|."""
    ref, _, reach = reference(q, k, v, table, context, drafts, bits, page, scale)
    norm = ref.norm()
    bound = 2.0 ** -19
    if q.dtype != F32:
        once = (ref.to(q.dtype).double() - ref).norm() / norm
        term = 2.0 ** -17 if q.dtype == BF16 else 2.0 ** -21
        bound = bound + 1.05 * once + term * reach.norm() / norm
    error = (out.double() - ref).norm() / norm
    assert error <= bound, (float(error), float(bound))


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("n,heads,kv,page", [
    (2, 6, 6, 16), (4, 4, 2, 13), (5, 6, 2, 16), (16, 2, 2, 7),      # up to 8 and 16 rows
    (9, 6, 2, 16), (30, 3, 3, 7),                                    # up to 32
    (16, 8, 2, 16), (24, 8, 2, 5), (40, 6, 6, 24), (33, 16, 2, 16)])  # more, several blocks
def test_errors_by_their_norm(cuda_device, ops, act, cache, dim, n, heads, kv, page):  # noqa: F811
    g = gen(100 * n + heads)
    k, v, table = make_cache([c + n for c in CONTEXTS], kv, dim, page, cache, "token", g)
    q = torch.randn(3, n, heads, dim, generator=g, device="cuda").to(act)
    bits = tree_bits(3, n, dim + n)
    out, _ = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits))
    norm_check(q, k, v, table, CONTEXTS, [n] * 3, bits, page, out, dim ** -0.5)


@pytest.mark.parametrize("act,cache,n", [(BF16, BF16, 4), (BF16, BF16, 64), (F16, F16, 64)])
def test_errors_of_a_split_sequence(cuda_device, ops, act, cache, n):  # noqa: F811
    """30,000 tokens, whose keys every CTA has a part of."""
    g = gen(n)
    k, v, table = make_cache([30000 + n], 2, 128, 64, cache, "token", g)
    q = torch.randn(1, n, 8, 128, generator=g, device="cuda").to(act)
    out, _ = ops.tree_attention(q, k, v, table, ints([30000]))
    norm_check(q, k, v, table, [30000], [n], None, 64, out, 128 ** -0.5)


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("heads", [2, 16])
def test_one_token_of_the_caches_type_is_paged_attention(cuda_device, ops, kind, heads):  # noqa: F811
    """Both keep two terms of the weights, so that the results differ where a rounding
    falls on another side: by a step of O, in few of its elements."""
    lens, g = [1, 17, 300, 2000], gen(heads)
    k, v, table = make_cache(lens, 1, 64, 16, kind, "token", g)
    q = torch.randn(4, heads, 64, generator=g, device="cuda").to(kind)
    a, _ = ops.paged_attention(q, k, v, table, ints(lens))
    b, _ = ops.tree_attention(q[:, None], k, v, table, ints([n - 1 for n in lens]))
    off = (a != b[:, 0]).float().mean().item()
    # differences below 2^-16 (bf16), 2^-17 (f16: FP32 sums too) of the largest elements'
    # terms against steps of 2^-8 and 2^-11 of them: 1 in 16 of them is a wide bound
    assert off <= 1 / 16, off
    assert torch.allclose(a.double(), b[:, 0].double(), rtol=torch.finfo(kind).eps, atol=2.0 ** -13)
