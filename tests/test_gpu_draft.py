"""The speculative-decoding operators (tree attention, verification of drafts,
compaction and copies of cache pages) against plain 64-bit computations, at the
sizes, layouts and masks where they can go wrong."""
import math
import random

import pytest
import torch

from .test_gpu_decode import BF16, F16, F32, TYPES, gen, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from cuda_transformer import ops as o
    return o


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pack(bits):
    """bool [..., n] as int32 words [..., ceil(n / 32)]."""
    words = -(-bits.shape[-1] // 32)
    wide = torch.nn.functional.pad(bits, (0, 32 * words - bits.shape[-1])).unflatten(-1, (words, 32))
    value = (wide.long() << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(value >= 2 ** 31, value - 2 ** 32, value).int()


def tree_bits(batch, n, seed):
    """Ancestors of the nodes of random trees."""
    rng = random.Random(seed)
    bits = torch.zeros(batch, n, n, dtype=torch.bool)
    for b in range(batch):
        for i in range(n):
            if i:
                bits[b, i] = bits[b, rng.randrange(max(0, i - 4), i)]
            bits[b, i, i] = True
    return bits.cuda()


# --------------------------------------------------------------- tree attention
def reference(q, k, v, table, context, drafts, bits, page, scale):
    """O, L and sum_j w_j |v_j| in 64 bits; `bits` [batch, n, n] or None (a chain)."""
    batch, n, heads, dim = q.shape
    group = heads // k.shape[1]
    out, reach = (torch.zeros(batch, n, heads, dim, dtype=torch.float64, device="cuda")
                  for _ in range(2))
    lse = torch.full((batch, n, heads), -math.inf, dtype=torch.float64, device="cuda")
    for b, (c, m) in enumerate(zip(context, drafts)):
        if c < 0 or m <= 0:
            continue
        pages = table[b, :-(-(c + m) // page)].long()
        kk, vv = (x[pages].transpose(1, 2).flatten(0, 1)[:c + m].double() for x in (k, v))
        kk, vv = (x.repeat_interleave(group, 1) for x in (kk, vv))
        sees = (torch.ones(m, m, device="cuda").tril() > 0 if bits is None else bits[b, :m, :m])
        s = torch.einsum("ihd,jhd->ihj", q[b, :m].double(), kk) * scale
        s[..., c:] = s[..., c:].masked_fill(~sees[:, None], -math.inf)
        lse[b, :m] = torch.logsumexp(s, -1)
        w = torch.softmax(s, -1).nan_to_num(0.0)
        out[b, :m] = torch.einsum("ihj,jhd->ihd", w, vv)
        reach[b, :m] = torch.einsum("ihj,jhd->ihd", w, vv.abs())
    return out, lse, reach


def check(q, k, v, table, context, drafts, bits, page, got, scale):
    """Tolerance.  A score's FP32 error is below 2^-21 |scale| sum|q_d k_d|; it moves
    the weights by that much relatively, so O by twice it times max|v|, and the sum adds
    2^-21 max|v| of its own.  16-bit results round once at the end (half a step of |O|,
    with 2^-10 of that half for a sum next to a tie), and with 16-bit activations the
    weights may be rounded to the cache's type (half a step of each: of sum w|v|)."""
    out, lse = got
    ref_o, ref_l, reach = reference(q, k, v, table, context, drafts, bits, page, scale)
    top_k, top_v = (x[torch.isfinite(x)].double().abs().max().item() if
                    torch.isfinite(x).any() else 0.0 for x in (k, v))
    score = abs(scale) * q.double().norm(dim=-1).max().item() * top_k * q.shape[-1] ** 0.5
    ds = 2.0 ** -21 * max(score, 1.0)
    assert out.dtype == q.dtype and lse.dtype == F32
    assert torch.equal(torch.isneginf(lse), torch.isneginf(ref_l))
    there = ~torch.isneginf(ref_l)
    assert torch.count_nonzero(out[~there]) == 0
    if not there.any():
        return
    assert (lse.double() - ref_l)[there].abs().max().item() <= 2 * ds + 2.0 ** -22 * (
        ref_l[there].abs().max().item())
    bound = (2 * ds + 2.0 ** -21) * top_v
    if q.dtype != F32:
        half = torch.finfo(q.dtype).eps / 2
        # (an f16 result below 2^-14 has steps of 2^-24; weights likewise)
        bound = bound + 1.001 * half * (ref_o.abs() + reach) + (2.0 ** -24 if q.dtype == F16 else 0)
    worst = ((out.double() - ref_o).abs() - bound).max().item()
    assert worst <= 0, worst


CONTEXTS = [0, 1, 2, 15, 16, 17, 40, 63, 64, 65, 129, 300, 1000]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("n,heads,kv,page,layout", [(8, 4, 4, 16, "head"), (5, 8, 1, 7, "token"),
                                                    (33, 16, 2, 64, "joint"), (1, 5, 1, 1, "head")])
def test_attention(cuda_device, ops, act, cache, dim, n, heads, kv, page, layout):
    """Trees of different sizes after contexts of different lengths."""
    g = gen(heads * 1000 + dim)
    drafts = [n if i % 3 else (5 * i) % n + 1 for i in range(len(CONTEXTS))]
    k, v, table = make_cache([c + m for c, m in zip(CONTEXTS, drafts)], kv, dim, page, cache,
                             layout, g)
    q = torch.randn(len(CONTEXTS), n, heads, dim, generator=g, device="cuda").to(act)
    bits = tree_bits(len(CONTEXTS), n, dim + n)
    got = ops.tree_attention(q, k, v, table, ints(CONTEXTS), ints(drafts), pack(bits))
    check(q, k, v, table, CONTEXTS, drafts, bits, page, got, dim ** -0.5)


@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 8, 16, 17, 31, 32, 64, 65, 100, 257])
@pytest.mark.parametrize("heads,kv,act,cache", [(1, 1, F32, F32), (6, 3, F32, BF16),
                                                (12, 1, BF16, BF16), (8, 2, F16, F16)])
def test_attention_chains(cuda_device, ops, n, heads, kv, act, cache):
    """Without a mask token i sees those up to itself (a piece of a prompt)."""
    context, g = [70, 0, 513], gen(heads + n)
    k, v, table = make_cache([c + n for c in context], kv, 64, 16, cache, "token", g)
    q = torch.randn(3, n, heads, 64, generator=g, device="cuda").to(act)
    got = ops.tree_attention(q, k, v, table, ints(context))
    check(q, k, v, table, context, [n] * 3, None, 16, got, 0.125)


@pytest.mark.parametrize("context", [[20000], [4096, 1], [1] * 200, [0] * 5, [9000, 0, 0, 33],
                                     [(7 * i * i) % 400 for i in range(200)] + [2000]])
@pytest.mark.parametrize("kv,group,n,cache", [(1, 8, 4, F16), (3, 2, 13, F32), (2, 4, 40, BF16)])
def test_attention_lengths(cuda_device, ops, context, kv, group, n, cache):
    """Few long rows (the length is split over the GPU), many short ones, none."""
    g = gen(len(context) + kv)
    k, v, table = make_cache([c + n for c in context], kv, 64, 32, cache, "head", g)
    q = torch.randn(len(context), n, kv * group, 64, generator=g, device="cuda").to(cache)
    bits = tree_bits(len(context), n, 1)
    got = ops.tree_attention(q, k, v, table, ints(context), mask=pack(bits))
    check(q, k, v, table, context, [n] * len(context), bits, 32, got, 0.125)


@pytest.mark.parametrize("kind,dim,n", [(F16, 64, 3), (F16, 64, 40), (BF16, 128, 33), (F32, 64, 2)])
def test_attention_long_shares(cuda_device, ops, kind, dim, n):
    """So many keys that every CTA goes through thousands of them in one piece: many
    sequences over the same pages.  All weights near 1: a sum that loses its low bits
    on the way shows."""
    batch, context, g = 56, 60000, gen(n)
    k, v, table = make_cache([context + n], 1, dim, 64, kind, "head", g)
    v += 1
    table = table.expand(batch, table.shape[1])
    q = (0.1 * torch.randn(batch, n, 1, dim, generator=g, device="cuda")).to(kind)
    out, lse = ops.tree_attention(q, k, v, table, ints([context] * batch))
    for b in (0, 17, batch - 1):
        one = slice(b, b + 1)
        check(q[one], k, v, table[one], [context], [n], None, 64, (out[one], lse[one]), dim ** -0.5)


@pytest.mark.parametrize("act,cache", TYPES)
def test_attention_masks(cuda_device, ops, act, cache):
    """Rows that see nothing of the draft, and without a context nothing at all;
    any bits (later tokens too); bits behind the draft; one mask for all sequences."""
    n, context, drafts, g = 35, [0, 0, 100, 31], [35, 10, 35, 33], gen(7)
    k, v, table = make_cache([c + m for c, m in zip(context, drafts)], 2, 64, 16, cache, "head", g)
    q = torch.randn(4, n, 4, 64, generator=g, device="cuda").to(act)
    bits = (torch.rand(1, n, n, generator=g, device="cuda") < 0.2).expand(4, n, n)
    bits = bits.clone()
    bits[:, ::4] = False
    bits[:, 1::4] = True
    bits = bits[:1].expand(4, n, n)
    mask = pack(bits[:1]).expand(4, n, 2)
    got = ops.tree_attention(q, k, v, table, ints(context), ints(drafts), mask)
    check(q, k, v, table, context, drafts, bits, 16, got, 0.125)
    wide = torch.full((4, n, 5), -1, dtype=torch.int32, device="cuda")[:, :, ::2]
    wide.copy_(torch.nn.functional.pad(pack(bits), (0, 1), value=-1))  # more words, strided
    again = ops.tree_attention(q, k, v, table, ints(context), ints(drafts), wide)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("cache", [F32, F16, BF16])
def test_attention_large_scores(cuda_device, ops, cache):
    """Scores of hundreds, one key far above the rest, late and early; a negative and
    a zero scale."""
    n, context, g = 6, [777, 777], gen(9)
    k, v, table = make_cache([c + n for c in context], 2, 128, 16, cache, "head", g)
    q = 8.0 * torch.randn(2, n, 8, 128, generator=g, device="cuda")
    for b, j in ((0, 770), (1, 3)):
        k[int(table[b, j // 16]), :, j % 16] = q[b, 2, ::4].to(cache)
    for scale in (128 ** -0.5, 1.0, -0.3, 0.0):
        got = ops.tree_attention(q, k, v, table, ints(context), scale=scale)
        check(q, k, v, table, context, [n, n], None, 16, got, scale)


def test_attention_sequences_that_take_no_part(cuda_device, ops):
    """Negative contexts and drafts of no tokens: zero rows, and nothing is read; draft
    lengths beyond the rows count as all of them."""
    n, g = 4, gen(11)
    k, v, table = make_cache([20, 24, 30, 40], 2, 64, 16, BF16, "token", g)
    table[1] = -1
    table[2] = 10 ** 9
    q = torch.randn(4, n, 4, 64, generator=g, device="cuda").to(BF16)
    out, lse = ops.tree_attention(q, k, v, table, ints([16, -1, 26, 36]), ints([9, 4, 0, -3]))
    assert torch.count_nonzero(out[1:]) == 0 and torch.isneginf(lse[1:]).all()
    check(q[:1], k, v, table[:1], [16], [4], None, 16, (out[:1], lse[:1]), 0.125)


@pytest.mark.parametrize("there", [[0, 299], [31, 32, 33, 290], [64], [5, 150, 151, 298, 299], []])
@pytest.mark.parametrize("n,cache", [(4, F32), (5, F16), (24, BF16)])
def test_attention_in_padded_batches(cuda_device, ops, there, n, cache):
    """300 places for sequences of which few are there, far apart (some long enough to be
    split); the others' table rows name no pages."""
    context = [-1] * 300
    for i, b in enumerate(there):
        context[b] = (1900, 3, 0, 700, 65)[i]
    g = gen(n)
    k, v, table = make_cache([max(c, 0) + n if c >= 0 else 0 for c in context], 2, 64, 16, cache,
                             "token", g)
    table = torch.where(ints(context)[:, None] >= 0, table, -1)
    if table.shape[1] < 121:  # a table that is split
        table = torch.nn.functional.pad(table, (0, 121 - table.shape[1]), value=-1)
    q = torch.randn(300, n, 4, 64, generator=g, device="cuda").to(cache)
    got = ops.tree_attention(q, k, v, table, ints(context))
    check(q, k, v, table, context, [n] * 300, None, 16, got, 0.125)


@pytest.mark.parametrize("act,cache,dim", [(BF16, BF16, 64), (F16, F16, 128), (F32, F16, 64)])
@pytest.mark.parametrize("n,context", [(300, [600, 40]), (602, [500])])
def test_attention_of_more_rows_than_a_wave(cuda_device, ops, act, cache, dim, n, context):
    """A piece of a prompt on 64 heads that share one: 150 and 301 blocks of 128 rows."""
    g = gen(n)
    k, v, table = make_cache([c + n for c in context], 1, dim, 16, cache, "head", g)
    table = torch.nn.functional.pad(table, (0, 4), value=-1)
    q = torch.randn(len(context), n, 64, dim, generator=g, device="cuda").to(act)
    got = ops.tree_attention(q, k, v, table, ints(context))
    check(q, k, v, table, context, [n] * len(context), None, 16, got, dim ** -0.5)


@pytest.mark.parametrize("n", [5, 40])
def test_attention_bad_lengths_and_pages(cuda_device, ops, n):
    """A length beyond the table, a page outside the cache: NaN in that sequence's rows
    alone."""
    context, g = [40, 50, 600, 70, 20], gen(5)
    k, v, table = make_cache([c + n for c in context], 2, 64, 16, F32, "head", g)
    q = torch.randn(5, n, 4, 64, generator=g, device="cuda")
    given, broken = [40, table.shape[1] * 16 - n + 1, 600, 70, 2 ** 31 - 1], table.clone()
    broken[2, 3] = k.shape[0]
    broken[3, (70 + n - 1) // 16] = -7
    lens = [n, n, n, n - 1 if n > 10 else n, n]
    out, lse = ops.tree_attention(q, k, v, broken, ints(given), ints(lens))
    for b in (1, 2, 3, 4):
        assert out[b, :lens[b]].isnan().all() and lse[b, :lens[b]].isnan().all()
        assert torch.count_nonzero(out[b, lens[b]:]) == 0
    check(q[:1], k, v, table[:1], [40], [n], None, 16, (out[:1], lse[:1]), 0.125)


def test_attention_without_pages(cuda_device, ops):
    k = torch.zeros(0, 2, 8, 64, device="cuda")
    q = torch.ones(2, 3, 4, 64, device="cuda")
    for table in (torch.zeros(2, 4, dtype=torch.int32, device="cuda"),
                  torch.zeros(2, 0, dtype=torch.int32, device="cuda")):
        out, lse = ops.tree_attention(q, k, k.clone(), table, ints([0, 5]), ints([0, 2]))
        assert torch.count_nonzero(out[0]) == 0 and torch.isneginf(lse[0]).all()
        assert out[1, :2].isnan().all() and torch.count_nonzero(out[1, 2]) == 0
    assert ops.tree_attention(q[:0], k, k, table[:0], ints([]))[0].shape == (0, 3, 4, 64)
    assert ops.tree_attention(q[:, :0], k, k, table, ints([1, 2]))[1].shape == (2, 0, 4)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("n,heads", [(6, 4), (40, 16)])
def test_attention_values_that_are_not_finite(cuda_device, ops, act, cache, n, heads):
    """A drafted token's NaN and infinities reach the rows that see it, and no others;
    a context token's all rows."""
    context, g = [33, 200, 64], gen(13)
    k, v, table = make_cache([c + n for c in context], 2, 64, 16, cache, "head", g)
    q = torch.randn(3, n, heads, 64, generator=g, device="cuda").to(act)
    bits = torch.eye(n, dtype=torch.bool, device="cuda").repeat(3, 1, 1)
    bits[:, :, 0] = True
    want = ops.tree_attention(q, k, v, table, ints(context), mask=pack(bits))
    dirty_k, dirty_v = k.clone(), v.clone()

    def put(cache, b, position, values):
        cache[int(table[b, position // 16]), :, position % 16] = values

    put(dirty_k, 0, 33 + 3, math.nan)                  # seen by row 3 of sequence 0
    put(dirty_v, 1, 200 + 2, math.inf)                 # by row 2 of sequence 1
    put(dirty_v, 1, 200 + 4, math.nan)                 # by row 4
    row = torch.zeros(64, dtype=cache, device="cuda")
    row[5] = -math.inf
    put(dirty_v, 2, 10, row)                           # by all of sequence 2
    out, lse = ops.tree_attention(q, dirty_k, dirty_v, table, ints(context), mask=pack(bits))
    assert out[0, 3].isnan().all() and lse[0, 3].isnan().all()
    assert not out[1, 2].isfinite().any() and out[1, 4].isnan().all()
    assert not out[2, ..., 5].isfinite().any() and out[2, ..., :5].isfinite().all()
    clean = torch.ones(3, n, dtype=torch.bool, device="cuda")
    clean[0, 3] = clean[1, 2] = clean[1, 4] = clean[2] = False
    # (their sums are the same ones, but for a tile that is summed in another order)
    assert torch.allclose(out[clean].double(), want[0][clean].double(), rtol=2.0 ** -7, atol=2e-3)
    assert torch.equal(lse[1], want[1][1]) and torch.equal(lse[2], want[1][2])


def test_attention_strided_query_and_far_pages(cuda_device, ops):
    """q as a view of a fused projection and with a stride along the head; pages more
    than 2^32 bytes and 2^31 elements into the cache."""
    g, n = gen(3), 3
    pages, page, kv, dim = 70000, 32, 8, 128   # 2.3e9 elements each
    context = [100, 28]
    table = torch.tensor([[69999, 0, 69990, 65537], [69000, -1, -1, -1]], dtype=torch.int32,
                         device="cuda")
    k, v = (torch.empty(pages, page, kv, dim, dtype=BF16, device="cuda").transpose(1, 2)
            for _ in range(2))
    for p in table.flatten().tolist():
        if p >= 0:
            for c in (k, v):
                c[p] = torch.randn(kv, page, dim, generator=g, device="cuda").to(BF16)
    qkv = torch.randn(2, n, 3, 24, dim, generator=g, device="cuda")
    used = table[table >= 0].long()
    t2 = torch.full_like(table, -1)
    t2[table >= 0] = torch.arange(used.numel(), device="cuda").int()
    turned = qkv[:, :, 2, :8].transpose(2, 3).contiguous().transpose(2, 3)
    for q in (qkv[:, :, 1, ::3], turned, qkv.to(BF16)[:, :, 0, :16]):
        got = ops.tree_attention(q, k, v, table, ints(context))
        check(q, k[used], v[used], t2, context, [n, n], None, page, got, dim ** -0.5)


def test_attention_of_one_token_is_paged_attention(cuda_device, ops):
    lens, g = [1, 17, 300, 0], gen(15)
    k, v, table = make_cache(lens, 2, 64, 16, BF16, "token", g)
    q = torch.randn(4, 8, 64, generator=g, device="cuda")
    a, la = ops.paged_attention(q, k, v, table, ints(lens))
    b, lb = ops.tree_attention(q[:, None], k, v, table, ints([n - 1 for n in lens]))
    assert (a - b[:, 0]).abs().max() <= 2e-6 and torch.equal(torch.isneginf(la), torch.isneginf(lb[:, 0]))


def test_attention_runs_alike_everywhere(cuda_device, ops):
    """The same bits run after run, on another stream, from a graph and beside another
    call that runs at the same time."""
    g, cases = gen(6), []
    for context, n, heads, kv, dim in (([5000, 3], 16, 8, 2, 128), ([64] * 40, 5, 4, 4, 32),
                                       ([30000], 64, 16, 1, 64), ([0], 3, 8, 8, 128)):
        k, v, table = make_cache([c + n for c in context], kv, dim, 64, BF16, "head", g)
        q = torch.randn(len(context), n, heads, dim, generator=g, device="cuda").to(BF16)
        c = ints(context)
        cases.append((q, k, v, table, c, ops.tree_attention(q, k, v, table, c)))
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in sides:
            with torch.cuda.stream(s):
                got.append([ops.tree_attention(*c[:5]) for c in cases])
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(x, y) for a, c in zip(r, cases) for x, y in zip(a, c[5]))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = [ops.tree_attention(*c[:5]) for c in cases]
        graphs.append((graph, held))
    for _ in range(2):
        for (graph, held), s in zip(graphs, sides):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(x, y) for a, c in zip(held, cases) for x, y in zip(a, c[5]))
            for a in held:
                a[0].zero_()


# ------------------------------------------------------------------ verification
def verified(target, tokens, parents, lens, drafter, uniform):
    """The definition, in Python floats (64 bits)."""
    batch, n, vocab = target.shape
    news, paths, counts = [], [], []
    for b in range(batch):
        m = n if lens is None else min(max(int(lens[b]), 0), n)
        path, new, node = [], [], 0 if m > 0 else None
        while node is not None:
            path.append(node)
            p = target[b, node].double().cpu()
            q = None if drafter is None else drafter[b, node].double().cpu()
            kids = [i for i in range(node + 1, m)
                    if (i - 1 if parents is None else int(parents[b, i])) == node
                    and 0 <= int(tokens[b, i]) < vocab]
            here, node, last = node, None, -1
            if uniform is None:
                if not p.isnan().any() and p.max() > -math.inf:
                    last = int((p == p.max()).nonzero()[0])
                node = next((i for i in kids if int(tokens[b, i]) == last), None)
            else:
                z = 1.0
                for i in kids:
                    x, u = int(tokens[b, i]), float(uniform[b, i])
                    if u * (1.0 if q is None else float(q[x])) * z < float(p[x]):
                        node = i
                        break
                    if q is None:
                        left = p.clone()
                        left[x] = 0.0
                        rest = z - float(p[x])
                    else:
                        left = (p / z - q).clamp(min=0.0)
                        rest = float(left.sum())
                    if rest > 0:
                        p, z = left, rest
                if node is None and p.sum() > 0:
                    upto = p.cumsum(0)
                    over = (upto > float(uniform[b, 0]) * upto[-1]).nonzero()
                    last = int(over[0]) if len(over) else int((p > 0).nonzero()[-1])
            new.append(last if node is None else int(tokens[b, node]))
        news.append(new + [-1] * (n - len(new)))
        paths.append(path + [-1] * (n - len(path)))
        counts.append(len(path))
    return torch.tensor(news), torch.tensor(paths).int(), torch.tensor(counts).int()


def draft(batch, n, vocab, mode, seed, kind=F32, chain=False, near=0.7, wide=2.0):
    g, rng = gen(seed), random.Random(seed)
    logits = wide * torch.randn(batch, n, vocab, generator=g, device="cuda")
    parents = [[-1] + [i - 1 if chain else rng.randrange(max(0, i - 4), i) for i in range(1, n)]
               for _ in range(batch)]
    parents = ints(parents)
    noise = 1.5 * torch.randn(batch, n, vocab, generator=g, device="cuda")
    drafter = torch.softmax(logits + noise, -1).to(kind)
    rows = torch.arange(batch, device="cuda")[:, None]
    of = drafter[rows, parents.long().clamp(min=0)].float()
    tokens = torch.multinomial(of.flatten(0, 1), 1, generator=g).view(batch, n)
    if mode != "sample":
        hit = torch.rand(batch, n, generator=g, device="cuda") < near
        best = logits.argmax(-1).gather(1, parents.long().clamp(min=0))
        tokens = torch.where(hit, best, tokens)
    uniform = torch.rand(batch, n, generator=g, device="cuda")
    target = logits.to(kind) if mode == "greedy" else torch.softmax(logits, -1).to(kind)
    return (target, tokens, parents, drafter if mode == "sample" else None,
            None if mode == "greedy" else uniform)


def same(got, want):
    for a, b in zip(got, want):
        assert a.is_cuda and a.dtype == b.dtype and torch.equal(a.cpu(), b), (a, b)


@pytest.mark.parametrize("mode", ["sample", "lookup", "greedy"])
@pytest.mark.parametrize("batch,n,vocab,chain", [(1, 1, 7, False), (5, 9, 1, False), (3, 8, 65, True),
                                                 (40, 16, 257, False), (9, 40, 5003, False),
                                                 (2, 5, 50257, True), (3, 12, 100256, False)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_verify(cuda_device, ops, mode, batch, n, vocab, chain, kind):
    target, tokens, parents, drafter, uniform = draft(batch, n, vocab, mode, n + vocab, kind, chain)
    given = None if chain else parents
    got = ops.verify_drafts(target, tokens, given, None, drafter, uniform)
    same(got, verified(target, tokens, given, None, drafter, uniform))
    lens = ints([(5 * b) % (n + 2) - 1 for b in range(batch)])
    got = ops.verify_drafts(target, tokens, given, lens, drafter, uniform)
    same(got, verified(target, tokens, given, lens, drafter, uniform))


def test_verify_many_siblings(cuda_device, ops):
    """All nodes are children of the first (and many of them refused), and a chain of
    the most nodes that fit."""
    for n, star in ((100, True), (1024, False)):
        target, tokens, parents, drafter, uniform = draft(2, n, 300, "sample", n, wide=4.0)
        if star:
            parents = torch.zeros_like(parents)
            uniform[:, 1:] = 0.99
        for q in (drafter, None):
            got = ops.verify_drafts(target, tokens, parents, None, q, uniform)
            same(got, verified(target, tokens, parents, None, q, uniform))


def test_verify_layouts_and_bad_trees(cuda_device, ops):
    """Strided and broadcast operands; parents out of order or out of range and tokens
    outside the vocabulary: such nodes are not tried."""
    target, tokens, parents, drafter, uniform = draft(6, 10, 130, "sample", 3)
    parents[0, 3], parents[1, 4], parents[2, 5], parents[3, 2] = 3, -5, 9, 10 ** 9
    tokens[0, 1], tokens[4, 1], tokens[5, 2] = -1, 130, 2 ** 40
    want = verified(target, tokens, parents, None, drafter, uniform)
    same(ops.verify_drafts(target, tokens, parents, None, drafter, uniform), want)
    wide = torch.full((6, 11, 200), math.nan, device="cuda")
    wide[:, 1:, 3:133] = target
    turned = drafter.transpose(1, 2).contiguous().transpose(1, 2)
    same(ops.verify_drafts(wide[:, 1:, 3:133], tokens.t().contiguous().t(),
                           torch.stack([parents, parents], 2)[:, :, 1], None, turned, uniform), want)
    row = target[:1].expand(6, 10, 130)
    got = ops.verify_drafts(row, tokens, parents, None, drafter, uniform)
    same(got, verified(row, tokens, parents, None, drafter, uniform))


def test_verify_rows_without_a_token(cuda_device, ops):
    """No probability left, NaN, -inf everywhere: no next token; equal best scores: the
    lowest; a drafter that is the target itself: everything is kept."""
    target, tokens, parents, drafter, uniform = draft(4, 4, 70, "sample", 8, chain=True)
    for bad in (0.0, math.nan):
        broken = target.clone()
        broken[1, 0] = bad
        for q in (None, drafter):
            new, path, counts = ops.verify_drafts(broken, tokens, None, None, q, uniform)
            assert new[1].tolist() == [-1] * 4 and counts[1] == 1
    scores = torch.zeros(4, 2, 9000, device="cuda")
    scores[0, 0] = -math.inf
    scores[1, 0, 8000] = math.nan
    scores[2, 0, 5000:] = 3.0
    two = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    two[2, 1] = 5000
    new, path, counts = ops.verify_drafts(scores, two)
    assert new.tolist() == [[-1, -1], [-1, -1], [5000, 0], [0, 0]]
    assert path.tolist() == [[0, -1], [0, -1], [0, 1], [0, 1]] and counts.tolist() == [1, 1, 2, 2]
    new, path, counts = ops.verify_drafts(drafter, tokens, None, None, drafter, uniform)
    assert counts.tolist() == [4] * 4 and torch.equal(new[:, :3], tokens[:, 1:])


def test_verify_numbers_at_the_ends(cuda_device, ops):
    """0 keeps whatever has a probability and draws the first token that has one; the
    largest number below 1 draws the last, even where sums are rounded."""
    p = torch.zeros(2, 2, 40000, device="cuda")
    p[:, :, 3] = p[:, :, 39990] = 0.5
    tokens = torch.full((2, 2), 7, device="cuda")  # probability 0: refused
    u = torch.zeros(2, 2, device="cuda")
    u[1] = 1 - 2.0 ** -24
    new, _, counts = ops.verify_drafts(p, tokens, uniform=u)
    assert new.tolist() == [[3, -1], [39990, -1]] and counts.tolist() == [1, 1]
    tokens[:, 1] = 3
    new, _, _ = ops.verify_drafts(p, tokens, uniform=u)
    assert new.tolist() == [[3, 3], [39990, -1]]  # (with 0.5 refused, the rest has one token)


@pytest.mark.parametrize("certain", [False, True])
def test_verify_keeps_the_targets_distribution(cuda_device, ops, certain):
    """First tokens of many verifications: a count of N p +- 6 sqrt(N p (1 - p)) for each of
    8 tokens (a chance of 2e-9 each outside it)."""
    g, N, n, vocab = gen(17), 40000, 4, 8
    p, q = torch.softmax(torch.randn(2, vocab, generator=g, device="cuda"), -1)
    parents = ints([[-1, 0, 0, 0]]).expand(N, n)
    if certain:  # the three candidates are always these
        tokens = torch.tensor([[0, 2, 5, 1]], device="cuda").expand(N, n)
    else:
        tokens = torch.multinomial(q.expand(N, vocab), n, replacement=True, generator=g)
    target, drafter = (x.expand(N, n, vocab) for x in (p, q))
    uniform = torch.rand(N, n, generator=g, device="cuda")
    new, _, counts = ops.verify_drafts(target, tokens, parents, None,
                                       None if certain else drafter, uniform)
    got = torch.bincount(new[:, 0], minlength=vocab).double()
    p = p.double()
    assert bool(((got - N * p).abs() <= 6 * (N * p * (1 - p)).sqrt()).all())
    assert (counts == 2).any() and (counts == 1).any()


# -------------------------------------------------------------- compaction, copies
def caches_of(count, pages, heads, page, dim, kind, layout, g):
    """Caches of numbers that tell every element apart (mod a prime)."""
    made = []
    for i in range(count):
        shape = {"head": (pages, heads, page, dim), "token": (pages, page, heads, dim),
                 "joint": (pages, 2, heads, page, dim), "odd": (pages, heads, page, dim + 1)}[layout]
        t = torch.randint(0, 251, shape, generator=g, device="cuda").to(kind)
        made.append(t.transpose(1, 2) if layout == "token" else t[:, i % 2] if layout == "joint"
                    else t[..., 1:] if layout == "odd" else t)
    return made


def compacted(caches, table, context, keep, counts, page):
    want = [c.clone() for c in caches]
    pages = caches[0].shape[0]
    for b in range(table.shape[0]):
        for j in range(min(int(counts[b]), keep.shape[1])):
            src, dst = int(context[b]) + int(keep[b, j]), int(context[b]) + j
            if context[b] < 0 or src <= dst or src >= table.shape[1] * page:
                continue
            ps, pd = int(table[b, src // page]), int(table[b, dst // page])
            if 0 <= ps < pages and 0 <= pd < pages:
                for w, c in zip(want, caches):
                    w[pd, :, dst % page] = c[ps, :, src % page]
    return want


@pytest.mark.parametrize("kind,layout,dim", [(F32, "head", 64), (BF16, "token", 128),
                                             (F16, "joint", 32), (BF16, "odd", 64),
                                             (F32, "odd", 7), (F16, "head", 3)])
@pytest.mark.parametrize("n,page", [(1, 4), (5, 1), (16, 16), (64, 7), (65, 16), (400, 13)])
def test_compact(cuda_device, ops, kind, layout, dim, n, page):
    g, rng = gen(n + dim), random.Random(n)
    context = [0, 3, 30, 17, 0, 9]
    counts, keep = [], torch.full((6, n), -1, dtype=torch.int32)
    for b, share in enumerate((0.5, 0.2, 1.0, 0.9, 0.0, 0.6)):
        rows = [i for i in range(n) if rng.random() < share]
        keep[b, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
        counts.append(len(rows))
    if n > 2:  # the last one alone, the longest way up; all but the first
        keep[3, 0], counts[3] = n - 1, 1
        keep[5, :n - 1], counts[5] = torch.arange(1, n).int(), n - 1
    width = -(-(30 + n) // page)
    caches = caches_of(3, 6 * width + 2, 2, page, dim, kind, layout, g)
    table = torch.randperm(6 * width + 2, generator=g, device="cuda")[:6 * width].view(6, width).int()
    want = compacted(caches, table, context, keep, counts, page)
    ops.kv_compact_(caches, table, ints(context), keep.cuda(), ints(counts))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


@pytest.mark.parametrize("n", [8, 200])
def test_compact_leaves_out_what_has_no_place(cuda_device, ops, n):
    """Sequences that take no part, pages out of range, positions behind the table,
    counts beyond the row; nothing else changes."""
    g = gen(n)
    width = 2 + n // 4
    caches = caches_of(2, 5 * width, 2, 4, 64, BF16, "token", g)
    table = torch.arange(5 * width, device="cuda").view(5, width).int()
    table[1, 1], table[2, 1], table[2, 0] = -1, 5 * width, 2 ** 31 - 1
    keep = torch.arange(1, n + 1).int().repeat(5, 1)
    context, counts = [-1, 1, 0, 4 * width - n + 3, 2], [n, n, n, n, n + 100]
    want = compacted(caches, table, context, keep, counts, 4)
    ops.kv_compact_(caches, table, ints(context), keep.cuda(), ints(counts))
    for c, w in zip(caches, want):
        assert torch.equal(c, w)
    # no order: nothing outside the draft's slots is touched
    before = [c.clone() for c in caches]
    wild = torch.randint(-3, n + 3, (5, n), generator=g, device="cuda").int()
    ops.kv_compact_(caches, table, ints([-1, -1, -1, -1, 2]), wild, ints([n] * 5))
    for c, w in zip(caches, before):
        assert torch.equal(c[:4 * width], w[:4 * width])


@pytest.mark.parametrize("layout,dim,kind", [("head", 64, F32), ("token", 128, BF16),
                                             ("joint", 64, F16), ("odd", 64, BF16), ("odd", 5, F32)])
@pytest.mark.parametrize("count,page", [(0, 4), (1, 1), (3, 16), (50, 13), (200, 128)])
def test_copy_pages(cuda_device, ops, layout, dim, kind, count, page):
    g = gen(count + dim)
    caches = caches_of(4, 2 * count + 5, 3, page, dim, kind, layout, g)
    pages = torch.randperm(2 * count + 5, generator=g, device="cuda").int()
    src, dst = pages[:count].clone(), pages[count:2 * count].clone()
    want = [c.clone() for c in caches]
    if count > 2:
        src[1], dst[2] = -1, 2 * count + 5
    for w, c in zip(want, caches):
        for s, d in zip(src.tolist(), dst.tolist()):
            if 0 <= s < len(c) and 0 <= d < len(c):
                w[d] = c[s]
    ops.kv_copy_pages_(caches, src, dst)
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_moves_of_many_caches_and_far_pages(cuda_device, ops):
    """More caches than one launch takes; pages more than 2^31 elements into a cache."""
    g = gen(2)
    caches = caches_of(131, 9, 2, 4, 32, BF16, "head", g)
    want = [c.clone() for c in caches]
    for w in want:
        w[7], w[8] = w[2], w[0]
    ops.kv_copy_pages_(caches, ints([2, 0]), ints([7, 8]))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    table = torch.arange(9, device="cuda").view(1, 9).int()
    want = compacted(caches, table, [3], torch.tensor([[2, 9, 20]]), [3], 4)
    ops.kv_compact_(caches, table, ints([3]), ints([[2, 9, 20]]), ints([3]))
    assert all(torch.equal(c, w) for c, w in zip(caches, want))
    big = torch.zeros(70000, 8, 32, 128, dtype=BF16, device="cuda")
    big[69999] = torch.randn(8, 32, 128, generator=g, device="cuda").to(BF16)
    ops.kv_copy_pages_([big], ints([69999]), ints([69997]))
    assert torch.equal(big[69997], big[69999]) and torch.count_nonzero(big[69998]) == 0
    table = ints([[69999, 69998]])
    keep = torch.arange(0, 32, 3, device="cuda").int()[None]
    kept = big[69999, :, ::3].clone()
    ops.kv_compact_([big], table, ints([0]), keep, ints([11]))
    assert torch.equal(big[69999, :, :11], kept)


def test_moves_are_captured(cuda_device, ops):
    """Verification and compaction in a graph: no value goes through the host."""
    target, tokens, parents, drafter, uniform = draft(4, 8, 300, "sample", 5)
    caches = caches_of(2, 20, 2, 4, 64, F32, "head", gen(5))
    table = torch.arange(20, device="cuda").view(4, 5).int()
    context = ints([0, 3, 7, 11])
    start = [c.clone() for c in caches]
    new, path, counts = verified(target, tokens, parents, None, drafter, uniform)
    want = compacted(caches, table, context.tolist(), path, counts, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.verify_drafts(target, tokens, parents, None, drafter, uniform)
        ops.kv_compact_(caches, table, context, got[1], got[2])
    for _ in range(2):
        for c, s in zip(caches, start):
            c.copy_(s)
        graph.replay()
        same(got, (new, path, counts))
        assert all(torch.equal(c, w) for c, w in zip(caches, want))


# ------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("act,cache", [(F32, F32), (F32, BF16), (BF16, BF16)])
def test_append_with_other_angles(cuda_device, ops, interleaved, act, cache):
    """Written where `positions` say, turned by `rotary_positions`: the same values as an
    append at those positions gives."""
    g = gen(21)
    cos, sin = ops.rotary_tables(50, 64, device="cuda")
    k, v = (torch.randn(6, 2, 64, generator=g, device="cuda").to(act) for _ in range(2))
    q = torch.randn(6, 4, 64, generator=g, device="cuda").to(act)
    slots, angles = ints([10, 11, 12, -1, 14, 15]), ints([10, 11, 11, 3, 50, -2])
    seq = ints([0] * 6)
    table = torch.arange(16, device="cuda").view(1, 16).int()
    kc, vc, other_k, other_v = (torch.zeros(16, 2, 4, 64, dtype=cache, device="cuda")
                                for _ in range(4))
    q1, k1 = ops.kv_append_(kc, vc, k, v, table, slots, seq_ids=seq, q=q, cos=cos, sin=sin,
                            interleaved=interleaved, want_k=True, rotary_positions=angles)
    for t, angle in ((0, 10), (1, 11), (2, 11)):
        one = slice(t, t + 1)
        q2, k2 = ops.kv_append_(other_k, other_v, k[one], v[one], table, ints([angle]), q=q[one],
                                seq_ids=seq[one], cos=cos, sin=sin, interleaved=interleaved,
                                want_k=True)
        assert torch.equal(q1[one], q2) and torch.equal(k1[one], k2)
        at, to = int(slots[t]), angle
        assert torch.equal(kc[at // 4, :, at % 4], other_k[to // 4, :, to % 4])
        assert torch.equal(vc[at // 4, :, at % 4], v[t].to(cache))
    assert torch.count_nonzero(q1[3]) == 0
    assert q1[4:].isnan().all() and k1[4:].isnan().all()      # no row of angles
    assert torch.count_nonzero(kc[3, :, 2:]) == 0
    # without a rotation the angles are not looked at
    ops.kv_append_(kc, vc, k, v, table, slots, seq_ids=seq, rotary_positions=angles)
    assert torch.equal(kc[3, :, 3], k[5].to(cache))


@pytest.mark.parametrize("kind", [F32, BF16])
def test_moves_of_single_elements(cuda_device, ops, kind):
    """A head dim of one, cut out of a wider row: its stride means nothing."""
    g = gen(31)
    wide = [torch.randint(0, 251, (6, 2, 4, 8), generator=g, device="cuda").to(kind) for _ in range(2)]
    want = [w.clone() for w in wide]
    caches = [w[..., 3::8] for w in wide]
    assert caches[0].shape[3] == 1 and caches[0].stride(3) == 8
    for w in want:
        w[5, ..., 3] = w[1, ..., 3]
        w[0, :, 1, 3] = w[0, :, 2, 3]
    ops.kv_copy_pages_(caches, ints([1]), ints([5]))
    ops.kv_compact_(caches, ints([[0]]), ints([0]), ints([[0, 2]]), ints([2]))
    assert all(torch.equal(w, x) for w, x in zip(wide, want))
