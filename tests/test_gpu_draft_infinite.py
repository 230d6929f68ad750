"""tree_attention over cached keys and values that are infinite: the formula's results, as
from paged_attention."""
import math

import pytest
import torch

from .test_gpu_decode import TYPES, gen, make_cache
from .test_gpu_draft import check, ints, ops, pack  # noqa: F401

pytestmark = pytest.mark.gpu

CONTEXTS, PAGE = [9, 100, 3000], 16
# up to 8, 16 and 32 rows, more, several blocks of rows
SHAPES = [(1, 4, 2), (3, 4, 2), (5, 6, 2), (9, 6, 2), (12, 8, 2), (40, 16, 2)]


def infinite_case(act, cache, n, heads, kv, dim, seed):
    """Sequences of one tile, of several and of several CTAs' shares; q is positive in dim
    3, so that an infinite key there decides the sign."""
    g = gen(seed)
    k, v, table = make_cache([c + n for c in CONTEXTS], kv, dim, PAGE, cache, "token", g)
    q = torch.randn(3, n, heads, dim, generator=g, device="cuda")
    q[..., 3] = q[..., 3].abs() + 0.1
    return k, v, table, q.to(act)


def slot(table, b, j):
    return int(table[b, j // PAGE]), slice(None), j % PAGE


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("n,heads,kv", SHAPES)
def test_infinite_keys(cuda_device, ops, act, cache, dim, n, heads, kv):  # noqa: F811
    """A key whose score is -inf has no weight, wherever it lies; one whose score is +inf
    leaves no number in the rows that see it."""
    k, v, table, q = infinite_case(act, cache, n, heads, kv, dim, dim + n)
    clean_k, keep = k.clone(), [torch.ones(c, dtype=torch.bool) for c in CONTEXTS]
    for b, c in enumerate(CONTEXTS):
        for j in (0, c // 2, c - 1):
            k[slot(table, b, j)][..., 3] = -math.inf
            keep[b][j] = False
    got = ops.tree_attention(q, k, v, table, ints(CONTEXTS))
    left = [int(x.sum()) for x in keep]  # the same without those keys
    k2, v2, table2 = make_cache([c + n for c in left], kv, dim, PAGE, cache, "head", gen(1))
    for b, (c, x) in enumerate(zip(CONTEXTS, keep)):
        for i, j in enumerate(x.nonzero()[:, 0].tolist() + list(range(c, c + n))):
            for new, old in ((k2, clean_k), (v2, v)):
                new[slot(table2, b, i)] = old[slot(table, b, j)]
    check(q, k2, v2, table2, left, [n] * 3, None, PAGE, got, dim ** -0.5)
    k[slot(table, 1, 50)][..., 3] = math.inf
    k[slot(table, 2, 3000 + n // 2)][..., 3] = math.inf
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS))
    assert out[1].isnan().all() and out[2, n // 2:].isnan().all()
    assert torch.equal(out[0], got[0][0]) and torch.equal(out[2, :n // 2], got[0][2, :n // 2])
    assert torch.equal(lse[0], got[1][0]) and torch.equal(lse[2, :n // 2], got[1][2, :n // 2])


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("n,heads,kv", SHAPES)
def test_infinite_values(cuda_device, ops, act, cache, dim, n, heads, kv):  # noqa: F811
    """An infinite value with a weight makes its dim of the result infinite, two of opposite
    signs NaN; the other dims are untouched.  A drafted token's reaches the rows that see
    it.  Scores are kept within a few units, so that every weight is a normal number of
    each type."""
    k, v, table, q = infinite_case(act, cache, n, heads, kv, dim, 80 + dim + n)
    clean = v.clone()
    want = ops.tree_attention(q, k, v, table, ints(CONTEXTS))
    for b, c in enumerate(CONTEXTS):
        v[slot(table, b, 0)][..., 5] = math.inf
        v[slot(table, b, c - 1)][..., dim - 2] = -math.inf
        v[slot(table, b, c // 2)][..., dim // 2] = math.inf
        v[slot(table, b, c // 3)][..., dim // 2] = -math.inf
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS))
    assert torch.equal(lse, want[1])
    assert (out[..., 5] == math.inf).all() and (out[..., dim - 2] == -math.inf).all()
    assert out[..., dim // 2].isnan().all()
    rest = [d for d in range(dim) if d not in (5, dim - 2, dim // 2)]
    assert torch.equal(out[..., rest], want[0][..., rest])
    check(q, k, clean, table, CONTEXTS, [n] * 3, None, PAGE, want, dim ** -0.5)
    # beside infinities of the context, drafted ones: from their token on
    for b, c in enumerate(CONTEXTS):
        v[slot(table, b, c + n // 2)][..., 7] = -math.inf
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS))
    assert torch.equal(lse, want[1])
    assert (out[..., 5] == math.inf).all() and (out[:, n // 2:, :, 7] == -math.inf).all()
    assert out[:, :n // 2, :, 7].isfinite().all() and out[..., dim // 2].isnan().all()
    out[..., [5, 7, dim - 2, dim // 2]] = want[0][..., [5, 7, dim - 2, dim // 2]]
    check(q, k, clean, table, CONTEXTS, [n] * 3, None, PAGE, (out, lse), dim ** -0.5)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("n,heads,kv", SHAPES)
def test_infinite_values_of_small_weight(cuda_device, ops, act, cache, dim, n, heads, kv):  # noqa: F811
    """Weights down to 2^-98 of the largest (2^-21 over an f16 cache) still count."""
    least = -(21 if cache == torch.float16 else 98) * math.log(2)
    k, v, table, q = infinite_case(act, cache, n, heads, kv, dim, dim)
    k.zero_()
    q.zero_()
    q[..., 3] = 1.0
    for b, c in enumerate(CONTEXTS):
        for i in range(min(c - 1, 31)):  # token 1 + i: dim i
            at = slot(table, b, 1 + i + (c // 2 if c > 60 else 0))
            k[at][..., 3] = least * (i + 1) / 32
            v[at][..., i] = math.inf if i % 2 else -math.inf
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS), scale=1.0)
    for b, c in enumerate(CONTEXTS):
        m = min(c - 1, 31)
        assert (out[b, ..., 1:m:2] == math.inf).all() and (out[b, ..., 0:m:2] == -math.inf).all()
        assert out[b, ..., m:].isfinite().all() and lse[b].isfinite().all()


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("n,heads,kv", SHAPES[1:])
def test_large_values_that_are_not_seen(cuda_device, ops, act, cache, n, heads, kv):  # noqa: F811
    """The largest numbers of the type, under drafted tokens that only themselves see, and
    under context tokens whose scores are -inf, leave the other rows bit for bit alone."""
    k, v, table, q = infinite_case(act, cache, n, heads, kv, 64, 7)
    bits = torch.eye(n, dtype=torch.bool, device="cuda").repeat(3, 1, 1)
    bits[:, 1] = False  # row 1 sees the context alone
    for b, c in enumerate(CONTEXTS):
        k[slot(table, b, c // 2)][..., 3] = -math.inf
    want = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits))
    for b, c in enumerate(CONTEXTS):
        v[slot(table, b, c // 2)] = torch.finfo(cache).max
        for i in range(2, n):
            v[slot(table, b, c + i)] = torch.finfo(cache).max * (-1) ** (i // 2)
    out, lse = ops.tree_attention(q, k, v, table, ints(CONTEXTS), mask=pack(bits))
    assert torch.equal(out[:, :2], want[0][:, :2]) and torch.equal(lse, want[1])
