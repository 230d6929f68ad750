"""The token-generation operators (paged cache append, one-token attention,
logits processing) against plain 64-bit computations, at the sizes, layouts and
masks where they can go wrong."""
import math

import pytest
import torch

from . import ct_helpers as H

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]
# half a unit in the last place, relative, with a factor 2 for the operator's
# own FP32 rounding falling on the other side of a tie
ROUND = {F32: 0.0, BF16: 2.0 ** -8, F16: 2.0 ** -10}


@pytest.fixture(scope="module")
def ops():
    from cuda_transformer import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_cache(lens, kv, dim, page, kind, layout, g, spare=3):
    """A cache of normal values in scattered pages; what no token may read is
    NaN: unused pages, slots past a sequence's end.  Table entries past the end
    are -1."""
    need = [-(-n // page) for n in lens]
    width, pool = max(1, max(need)), sum(need) + spare
    perm = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    shape = {"head": (pool, kv, page, dim), "token": (pool, page, kv, dim),
             "joint": (pool, 2, kv, page, dim)}[layout]
    if layout == "joint":
        both = torch.full(shape, math.nan, device="cuda", dtype=kind)
        k, v = both[:, 0], both[:, 1]
    else:
        k, v = (torch.full(shape, math.nan, device="cuda", dtype=kind) for _ in range(2))
        if layout == "token":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        for i in range(need[b]):
            used = min(page, n - i * page)
            p = int(table[b, i])
            for c in (k, v):
                c[p, :, :used] = torch.randn(kv, used, dim, generator=g, device="cuda").to(kind)
    return k, v, table


def reference(q, k, v, table, lens, page, scale):
    batch, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(batch, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n <= 0:
            continue
        pages = table[b, :-(-n // page)].long()
        kk, vv = (c[pages].transpose(1, 2).flatten(0, 1)[:n].double() for c in (k, v))
        kk, vv = (t.repeat_interleave(group, 1) for t in (kk, vv))
        s = torch.einsum("hd,nhd->hn", q[b].double(), kk) * scale
        lse[b] = torch.logsumexp(s, -1)
        out[b] = torch.einsum("hn,nhd->hd", torch.softmax(s, -1), vv)
    return out, lse


def check_attention(q, k, v, table, lens, page, got, scale):
    """Tolerance: a score's FP32 error is below 2^-21 |scale| sum|q_d k_d|; it moves
    the weights by that much relatively, so O by twice it times max|v|, and
    the weighted sum adds 2^-21 max|v| of its own."""
    out, lse = got
    ref_o, ref_l = reference(q, k, v, table, lens, page, scale)
    live = k[torch.isfinite(k)]
    top_k = live.double().abs().max().item() if live.numel() else 0.0
    live = v[torch.isfinite(v)]
    top_v = live.double().abs().max().item() if live.numel() else 0.0
    reach = abs(scale) * q.double().norm(dim=-1).max().item() * top_k * q.shape[-1] ** 0.5
    ds = 2.0 ** -21 * max(reach, 1.0)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    assert torch.equal(torch.isneginf(lse), torch.isneginf(ref_l))
    there = ~torch.isneginf(ref_l)
    assert (lse.double() - ref_l)[there].abs().max().item() <= 2 * ds + 2.0 ** -22 * (
        ref_l[there].abs().max().item()) if there.any() else True
    bound = (2 * ds + 2.0 ** -21) * top_v + ROUND[q.dtype] * ref_o.abs()
    assert bool(((out.double() - ref_o).abs() <= bound).all())
    assert torch.count_nonzero(out[~there]) == 0


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 300, 0, 1000]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("heads,kv,page,layout", [(4, 4, 16, "head"), (8, 1, 7, "token"),
                                                  (32, 2, 64, "joint"), (5, 1, 1, "head")])
def test_attention(cuda_device, ops, act, cache, dim, heads, kv, page, layout):
    g = gen(heads * 1000 + dim)
    k, v, table = make_cache(LENGTHS, kv, dim, page, cache, layout, g)
    q = torch.randn(len(LENGTHS), heads, dim, generator=g, device="cuda").to(act)
    lens = torch.tensor(LENGTHS, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(q, k, v, table, lens)
    check_attention(q, k, v, table, LENGTHS, page, got, dim ** -0.5)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (6, 2), (12, 1), (17, 1), (24, 1), (64, 2),
                                      (7, 7)])
def test_attention_groups(cuda_device, ops, heads, kv):
    lens, g = [70, 0, 513], gen(heads)
    k, v, table = make_cache(lens, kv, 64, 16, BF16, "token", g)
    q = torch.randn(3, heads, 64, generator=g, device="cuda")
    got = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    check_attention(q, k, v, table, lens, 16, got, 0.125)


@pytest.mark.parametrize("lens", [[20000], [4096, 1], [1] * 300, [0] * 5, [9000, 0, 0, 33],
                                  [(7 * i * i) % 400 for i in range(300)] + [2000]])
@pytest.mark.parametrize("kv,group,cache", [(1, 8, F16), (3, 2, F32)])
def test_attention_lengths(cuda_device, ops, lens, kv, group, cache):
    """Few long rows (the length is split over the GPU), many short ones, none."""
    g = gen(len(lens) + kv)
    k, v, table = make_cache(lens, kv, 64, 32, cache, "head", g)
    q = torch.randn(len(lens), kv * group, 64, generator=g, device="cuda").to(cache)
    got = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    check_attention(q, k, v, table, lens, 32, got, 0.125)


@pytest.mark.parametrize("cache", [F32, F16])
def test_attention_large_scores(cuda_device, ops, cache):
    """Scores of hundreds, one key far above the rest, late in the sequence and
    early; a negative and a zero scale."""
    lens, g = [777, 777], gen(9)
    k, v, table = make_cache(lens, 2, 128, 16, cache, "head", g)
    q = 8.0 * torch.randn(2, 8, 128, generator=g, device="cuda")
    for b, j in ((0, 770), (1, 3)):
        k[int(table[b, j // 16]), :, j % 16] = q[b, ::4].to(cache)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for scale in (128 ** -0.5, 1.0, -0.3, 0.0):
        got = ops.paged_attention(q, k, v, table, n, scale=scale)
        check_attention(q, k, v, table, lens, 16, got, scale)


def test_attention_strided_query_and_far_pages(cuda_device, ops):
    """q as a view of a fused projection; pages more than 2^32 bytes and 2^31
    elements into the cache."""
    g = gen(3)
    pages, page, kv, dim = 70000, 32, 8, 128   # 2.3e9 elements each
    lens = [100, 31]
    table = torch.tensor([[69999, 0, 69990, 65537], [69000, -1, -1, -1]], dtype=torch.int32,
                         device="cuda")
    k, v = (torch.empty(pages, page, kv, dim, dtype=BF16, device="cuda").transpose(1, 2)
            for _ in range(2))
    for p in table.flatten().tolist():
        if p >= 0:
            for c in (k, v):
                c[p] = torch.randn(kv, page, dim, generator=g, device="cuda").to(BF16)
    qkv = torch.randn(2, 3, 24, dim, generator=g, device="cuda")
    q = qkv[:, 1, ::3]
    got = ops.paged_attention(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    used = table[table >= 0].long()
    small = torch.arange(used.numel(), device="cuda").int()
    t2 = torch.full_like(table, -1)
    t2[table >= 0] = small
    check_attention(q, k[used], v[used], t2, lens, page, got, dim ** -0.5)


def test_attention_bad_lengths_and_pages(cuda_device, ops):
    """A length beyond the table, a page outside the cache: NaN for that row
    alone.  A negative length counts as none."""
    lens, g = [40, 50, 60, 70, 20], gen(5)
    k, v, table = make_cache(lens, 2, 64, 16, F32, "head", g)
    q = torch.randn(5, 4, 64, generator=g, device="cuda")
    given = torch.tensor([40, table.shape[1] * 16 + 1, 60, 70, -3], dtype=torch.int32,
                         device="cuda")
    broken = table.clone()
    broken[2, 1] = k.shape[0]
    broken[3, 4] = -7
    out, lse = ops.paged_attention(q, k, v, broken, given)
    for b in (1, 2, 3):
        assert out[b].isnan().all() and lse[b].isnan().all()
    check_attention(q[[0, 4]], k, v, table[[0, 4]], [40, 0], 16, (out[[0, 4]], lse[[0, 4]]), 0.125)


def test_attention_without_pages(cuda_device, ops):
    """An empty pool and an empty table: nothing can be read."""
    k = torch.zeros(0, 2, 8, 64, device="cuda")
    q = torch.ones(2, 4, 64, device="cuda")
    lens = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    for table in (torch.zeros(2, 4, dtype=torch.int32, device="cuda"),
                  torch.zeros(2, 0, dtype=torch.int32, device="cuda")):
        out, lse = ops.paged_attention(q, k, k.clone(), table, lens)
        assert torch.count_nonzero(out[0]) == 0 and torch.isneginf(lse[0]).all()
        assert out[1].isnan().all() and lse[1].isnan().all()


def test_attention_workspace_is_reusable(cuda_device, ops):
    """One workspace over calls of different sizes; the same bits with a fresh
    one, run after run, on another stream and replayed from a graph."""
    g = gen(6)
    ws = ops.paged_attention_workspace(16, 1, 128)
    cases = []
    for lens, heads, kv, dim in (([5000, 3], 8, 2, 128), ([64] * 40, 4, 4, 32), ([30000], 16, 1, 64),
                                 ([0], 8, 8, 128)):
        k, v, table = make_cache(lens, kv, dim, 64, BF16, "head", g)
        q = torch.randn(len(lens), heads, dim, generator=g, device="cuda").to(BF16)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        cases.append((q, k, v, table, n, ops.paged_attention(q, k, v, table, n)))
    side = torch.cuda.Stream()
    for _ in range(3):
        for q, k, v, table, n, want in cases:
            got = ops.paged_attention(q, k, v, table, n, workspace=ws)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.paged_attention(*c[:5], workspace=ws) for c in cases]
    side.synchronize()
    assert all(torch.equal(a, b) for r, c in zip(got, cases) for a, b in zip(r, c[5]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [ops.paged_attention(*c[:5], workspace=ws) for c in cases]
    for _ in range(2):
        for r in held:
            r[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for r, c in zip(held, cases) for a, b in zip(r, c[5]))


# ------------------------------------------------------------------ append
def rotate(x, pos, cos, sin, interleaved):
    """64 bits: rows of x [n, heads, dim] turned by their positions' angles,
    and a bound on the FP32 error of doing it (four roundings of |a| + |b|)."""
    x = x.double()
    bound = torch.zeros_like(x)
    if cos is None:
        return x, bound
    hr = cos.shape[1]
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    ia, ib = ((slice(0, 2 * hr, 2), slice(1, 2 * hr, 2)) if interleaved
              else (slice(0, hr), slice(hr, 2 * hr)))
    a, b = x[..., ia].clone(), x[..., ib].clone()
    y = x.clone()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    bound[..., ia] = bound[..., ib] = 2.0 ** -22 * (a.abs() + b.abs())
    return y, bound


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv,dim,rot,page,layout,interleaved", [
    (4, 4, 64, 64, 16, "head", False), (8, 2, 128, 128, 16, "token", False),
    (3, 1, 32, 0, 5, "joint", False), (6, 3, 128, 32, 13, "token", True),
    (2, 2, 64, 64, 1, "head", True), (5, 1, 32, 6, 8, "head", False),
    (5, 5, 64, 10, 8, "token", True), (0, 2, 128, 64, 32, "head", False)])
def test_append(cuda_device, ops, act, cache, heads, kv, dim, rot, page, layout, interleaved):
    """Prompts and single tokens, in any order, into a cache whose other values
    stay as they were."""
    g = gen(dim + rot + heads)
    lens = [37, 1, 5, 0, 64]
    k_cache, v_cache, table = make_cache(lens, kv, dim, page, cache, layout, g)
    ids = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)]).int()
    pos = torch.cat([torch.arange(n) for n in lens]).int()
    order = torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))[:70]
    ids, pos = ids[order].cuda(), pos[order].cuda()
    qkv = torch.randn(70, heads + 2 * kv, dim, generator=g, device="cuda").to(act)
    q, k, v = qkv.split([heads, kv, kv], 1)
    cos, sin = ops.rotary_tables(64, rot, device="cuda") if rot else (None, None)
    want_k, want_v = k_cache.clone(), v_cache.clone()
    q_out, k_out = ops.kv_append_(k_cache, v_cache, k, v, table, pos, seq_ids=ids,
                                  q=q if heads else None, cos=cos, sin=sin,
                                  interleaved=interleaved, want_k=True)
    where = (table[ids.long(), pos.long() // page].long(), slice(None), pos.long() % page)
    kr, kb = rotate(k, pos, cos, sin, interleaved)
    got = k_cache[where].double()
    assert bool(((got - kr).abs() <= kb + ROUND[cache] * kr.abs() + 2.0 ** -25).all())
    assert bool(((k_out.double() - kr).abs() <= kb + ROUND[act] * kr.abs() + 2.0 ** -25).all())
    assert torch.equal(v_cache[where], v.to(cache))
    if heads:
        qr, qb = rotate(q, pos, cos, sin, interleaved)
        assert q_out.shape == q.shape and q_out.dtype == act
        assert bool(((q_out.double() - qr).abs() <= qb + ROUND[act] * qr.abs() + 2.0 ** -25).all())
    want_k[where], want_v[where] = k_cache[where], v_cache[where]
    assert torch.equal(k_cache.nan_to_num(7.0), want_k.nan_to_num(7.0))
    assert torch.equal(v_cache.nan_to_num(7.0), want_v.nan_to_num(7.0))


def test_append_odd_strides(cuda_device, ops):
    """Inputs at odd offsets and strides, a last stride other than one, and a
    cache with padded rows at an odd offset."""
    g = gen(11)
    pool = torch.zeros(4 * 2 * 8 * 37 + 1, dtype=F32, device="cuda")
    k_cache = pool[1:].view(4, 2, 8, 37)[..., 3:35]
    v_cache = k_cache.clone()
    table = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32, device="cuda")
    flat = torch.randn(2 * 3 * 33 + 1, generator=g, device="cuda")
    k = flat[1:].view(2, 3, 33)[:, :2, :32]
    v = torch.randn(32, 2, 2, generator=g, device="cuda").permute(1, 2, 0)
    pos = torch.tensor([9, 3], dtype=torch.int32, device="cuda")
    cos, sin = ops.rotary_tables(16, 32, device="cuda")
    _, k_out = ops.kv_append_(k_cache, v_cache, k, v, table, pos, cos=cos, sin=sin, want_k=True)
    kr, kb = rotate(k, pos, cos, sin, False)
    assert bool(((k_out.double() - kr).abs() <= kb).all())
    for t, (page, slot) in enumerate(((0, 1), (3, 3))):
        assert torch.equal(k_cache[page, :, slot], k_out[t])
        assert torch.equal(v_cache[page, :, slot], v[t])
    assert torch.count_nonzero(pool) == torch.count_nonzero(k_out)


def test_append_padding_and_bad_places(cuda_device, ops):
    """Padding tokens append nothing and give zeros; tokens with no place
    append nothing and give NaN."""
    g = gen(12)
    k_cache, v_cache = (torch.zeros(4, 2, 8, 64, device="cuda") for _ in range(2))
    table = torch.tensor([[2, 9], [-1, 1]], dtype=torch.int32, device="cuda")
    #       fine  pad  page 9  page -1  past the table  no sequence  no angle
    ids = torch.tensor([0, 0, 0, 1, 1, 2, 1, -1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, -1, 8, 2, 16, 0, 12, 0], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(8, 2, 64, generator=g, device="cuda") for _ in range(3))
    cos, sin = ops.rotary_tables(12, 64, device="cuda")
    q_out, k_out = ops.kv_append_(k_cache, v_cache, k, v, table, pos, seq_ids=ids, q=q, cos=cos,
                                  sin=sin, want_k=True)
    assert torch.equal(k_cache[2, :, 3], k_out[0]) and torch.equal(v_cache[2, :, 3], v[0])
    assert torch.count_nonzero(k_cache) == torch.count_nonzero(k_out[0])
    assert torch.count_nonzero(v_cache) == torch.count_nonzero(v[0])
    assert q_out[0].isfinite().all() and torch.count_nonzero(q_out[1]) == 0
    assert torch.count_nonzero(k_out[1]) == 0
    assert q_out[2:].isnan().all() and k_out[2:].isnan().all()


def test_append_far_pages_and_no_tokens(cuda_device, ops):
    g = gen(13)
    k_cache, v_cache = (torch.empty(70000, 32, 8, 128, dtype=BF16, device="cuda").transpose(1, 2)
                        for _ in range(2))
    table = torch.tensor([[69999]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, 8, 128, generator=g, device="cuda") for _ in range(2))
    pos = torch.tensor([31], dtype=torch.int32, device="cuda")
    ops.kv_append_(k_cache, v_cache, k, v, table, pos)
    assert torch.equal(k_cache[69999, :, 31], k[0].to(BF16))
    assert torch.equal(v_cache[69999, :, 31], v[0].to(BF16))
    q_out, _ = ops.kv_append_(k_cache, v_cache, k[:0], v[:0], table, pos[:0], q=k[:0])
    assert q_out.shape == (0, 8, 128)


def test_append_then_attend(cuda_device, ops):
    """Token by token through the cache is causal attention of the whole
    sequence (with rotary angles, grouped heads)."""
    g = gen(14)
    n, heads, kv, dim = 40, 6, 2, 64
    q, k, v = (torch.randn(2, n, h, dim, generator=g, device="cuda") for h in (heads, kv, kv))
    k_cache, v_cache = (torch.full((10, kv, 8, dim), math.nan, device="cuda") for _ in range(2))
    table = torch.randperm(10, generator=g, device="cuda").int().view(2, 5)
    cos, sin = ops.rotary_tables(n, dim, device="cuda")
    outs = []
    for j in range(n):
        pos = torch.full((2,), j, dtype=torch.int32, device="cuda")
        qr, _ = ops.kv_append_(k_cache, v_cache, k[:, j], v[:, j], table, pos, q=q[:, j], cos=cos,
                               sin=sin)
        outs.append(ops.paged_attention(qr, k_cache, v_cache, table, pos + 1)[0])
    got = torch.stack(outs, 1).double()
    at = torch.arange(n, device="cuda")
    for b in range(2):
        qd, kd = rotate(q[b], at, cos, sin, False)[0], rotate(k[b], at, cos, sin, False)[0]
        kd, vd = (t.repeat_interleave(heads // kv, 1) for t in (kd, v[b].double()))
        s = torch.einsum("nhd,mhd->hnm", qd, kd) * dim ** -0.5
        s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
        ref = torch.einsum("hnm,mhd->nhd", s.softmax(-1), vd)
        # a score's error 2^-21 |q||k| scale (~2^-17), twice, times max|v| (~4)
        assert (got[b] - ref).abs().max().item() <= 2.0 ** -14


# ------------------------------------------------------------------ logits
def logits_reference(x, tokens, lens, plens, rep, freq, pres, ids, values, mask):
    """64 bits, and a bound on the FP32 error: a rounding of 2^-23 for each of up to
    (4 + number of biases) operations on terms of the sizes summed here."""
    x = x.double().clone()
    rows, vocab = x.shape
    size, steps = x.abs().clone(), torch.full_like(x, 4.0)
    for r in range(rows):
        if tokens is not None:
            n = tokens.shape[1] if lens is None else min(max(int(lens[r]), 0), tokens.shape[1])
            m = 0 if plens is None else min(max(int(plens[r]), 0), n)

            def count(t):
                return t[(t >= 0) & (t < vocab)].bincount(minlength=vocab).double()

            seen, made = count(tokens[r, :n]) > 0, count(tokens[r, m:n])
            rr = 1.0 if rep is None else float(rep[r])
            ff = 0.0 if freq is None else float(freq[r])
            pp = 0.0 if pres is None else float(pres[r])
            x[r] = torch.where(seen, torch.where(x[r] > 0, x[r] / rr, x[r] * rr), x[r])
            size[r] = torch.maximum(size[r], x[r].abs()) + ff * made + abs(pp)
            x[r] -= ff * made + pp * (made > 0)
        if ids is not None:
            for i, w in zip(ids[r].tolist(), values[r].tolist()):
                if 0 <= i < vocab:
                    x[r, i] += w
                    size[r, i] += abs(w)
                    steps[r, i] += 1
        if mask is not None:
            bits = (mask[r][:, None] >> torch.arange(32, device=x.device)) & 1
            x[r].masked_fill_(bits.flatten()[:vocab] == 0, -math.inf)
    return x, 2.0 ** -23 * steps * size


def check_logits(got, *args):
    ref, bound = logits_reference(*args)
    assert got.dtype == F32 and got.shape == ref.shape
    bad = ~torch.isfinite(ref)
    assert torch.equal(got[bad].double(), ref[bad])
    assert bool(((got.double() - ref).abs() <= bound)[~bad].all())


def random_mask(rows, vocab, g, extra=0):
    return torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32) + extra), generator=g,
                         device="cuda").int()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocab,hist,bias", [(1, 1, 3, 2), (3, 65, 40, 5), (2, 8191, 300, 0),
                                                  (5, 8193, 9000, 40), (2, 50257, 1, 300),
                                                  (40, 20001, 1500, 20), (1, 2000, 2000, 3000),
                                                  (1, 100256, 500, 16), (4, 33000, 0, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_logits(cuda_device, ops, dtype, rows, vocab, hist, bias, masked):
    g = gen(vocab + rows)
    x = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    # ids outside the vocabulary (as padding has them) among the rest, many repeats
    tokens = torch.randint(-2, min(vocab, 200) + 2, (rows, hist), generator=g, device="cuda")
    lens = torch.randint(0, hist + 1, (rows,), generator=g, device="cuda").int()
    lens[0] = hist + 5                              # clamped to hist
    plens = torch.randint(-1, hist + 2, (rows,), generator=g, device="cuda").int()
    rep, freq, pres = (torch.rand(rows, generator=g, device="cuda") for _ in range(3))
    rep = rep + 0.6
    ids = values = None
    if bias:
        ids = torch.randint(-1, vocab + 1, (rows, bias), generator=g, device="cuda")
        ids[:, bias // 2:] = ids[:, :bias - bias // 2]   # tokens listed twice
        values = torch.randn(rows, bias, generator=g, device="cuda")
    mask = random_mask(rows, vocab, g) if masked else None
    got = ops.logits_process(x, tokens, lens, plens, rep, freq, pres, ids, values, mask)
    check_logits(got, x, tokens, lens, plens, rep, freq, pres, ids, values, mask)
    again = ops.logits_process(x, tokens, lens, plens, rep, freq, pres, ids, values, mask)
    assert torch.equal(got, again)


@pytest.mark.parametrize("rows,vocab,hist,bias", [(310, 700, 900, 4), (300, 60000, 20000, 0),
                                                  (300, 1001, 60, 700), (330, 40000, 40000, 400)])
@pytest.mark.parametrize("masked", [False, True])
def test_logits_more_rows_than_sms(cuda_device, ops, rows, vocab, hist, bias, masked):
    """Rows of which a block has several, whose tokens and biases fit its lists together, one
    by one, or not at all; histories beyond 16-bit counts.  A row's result is the same
    whichever rows it is computed with; some are compared with 64 bits."""
    g = gen(rows + vocab)
    x = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    tokens = torch.randint(-2, vocab + 2, (rows, hist), generator=g, device="cuda")
    tokens[::2] %= 90
    lens = torch.randint(0, hist + 1, (rows,), generator=g, device="cuda").int()
    plens = torch.randint(0, hist + 1, (rows,), generator=g, device="cuda").int()
    rep, freq, pres = (torch.rand(rows, generator=g, device="cuda") + 0.6 for _ in range(3))
    ids = values = None
    if bias:
        ids = torch.randint(-1, vocab + 1, (rows, bias), generator=g, device="cuda")
        ids[:, bias // 2:] = ids[:, :bias - bias // 2]
        values = torch.randn(rows, bias, generator=g, device="cuda")
    mask = random_mask(rows, vocab, g) if masked else None
    args = (x, tokens, lens, plens, rep, freq, pres, ids, values, mask)
    got = ops.logits_process(*args)
    some = list(range(0, rows, 47)) + [rows - 1]
    check_logits(got[some], *(None if a is None else a[some] for a in args))
    for r0 in range(0, rows, 110):
        part = ops.logits_process(*(None if a is None else a[r0:r0 + 110] for a in args))
        assert torch.equal(part, got[r0:r0 + 110])


def test_logits_a_great_many_rows(cuda_device, ops):
    g = gen(77)
    rows, vocab = 80000, 40
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    tokens = torch.randint(0, vocab, (rows, 9), generator=g, device="cuda")
    pres = torch.rand(rows, generator=g, device="cuda")
    got = ops.logits_process(x, tokens, presence=pres)
    seen = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens, True)
    ref = torch.where(seen, x.double() - pres.double()[:, None], x.double())
    # one rounding, of a term below 8
    assert bool(((got.double() - ref).abs() <= 2.0 ** -21).all())


@pytest.mark.parametrize("keep", ["nothing", "penalties", "bias", "mask"])
def test_logits_single_options(cuda_device, ops, keep):
    g = gen(21)
    x = torch.randn(3, 1001, generator=g, device="cuda")
    kw = {}
    if keep == "penalties":
        kw = {"tokens": torch.randint(0, 1001, (3, 50), generator=g, device="cuda"),
              "presence": torch.full((3,), -0.5, device="cuda")}
    elif keep == "bias":
        kw = {"bias_ids": torch.tensor([[5, 5, 7]] * 3, device="cuda"),
              "bias_values": torch.tensor([[1.0, 2.0, math.inf]] * 3, device="cuda")}
    elif keep == "mask":
        kw = {"mask": torch.zeros(3, 32, dtype=torch.int32, device="cuda")}
    got = ops.logits_process(x, **kw)
    names = ("tokens", "lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids",
             "bias_values", "mask")
    check_logits(got, x, *(kw.get(n) for n in names))


def test_logits_infinities_and_masks(cuda_device, ops):
    """-inf and the lowest FP32 value stay what they are; a masked NaN or +inf
    logit and a masked +inf bias come out -inf."""
    x = torch.tensor([[1.0, -math.inf, math.nan, math.inf, torch.finfo(F32).min, -2.0]],
                     device="cuda")
    tokens = torch.tensor([[1, 1, 4, 5]], device="cuda")
    mask = torch.tensor([[0b110011]], dtype=torch.int32, device="cuda")
    one = torch.ones(1, device="cuda")
    got = ops.logits_process(x, tokens, repetition=one, frequency=one, mask=mask,
                             bias_ids=torch.tensor([[3, 0]], device="cuda"),
                             bias_values=torch.tensor([[math.inf, 0.5]], device="cuda"))
    want = torch.tensor([[1.5, -math.inf, -math.inf, -math.inf, torch.finfo(F32).min, -3.0]],
                        device="cuda")
    assert torch.equal(got, want)


def test_logits_strides_and_streams(cuda_device, ops):
    """Rows at an odd stride and offset, operands shared by all rows, a
    transposed operand, another stream."""
    g = gen(23)
    rows, vocab = 6, 10007
    x = torch.randn(rows * 10010 + 1, generator=g, device="cuda")[1:].view(rows, 10010)[:, 2:2 + vocab]
    tokens = torch.randint(0, vocab, (400, rows), generator=g, device="cuda").t()
    rep = torch.full((1,), 1.3, device="cuda").expand(rows)
    ids = torch.randint(0, vocab, (1, 9), generator=g, device="cuda").expand(rows, 9)
    values = torch.randn(1, 9, generator=g, device="cuda").expand(rows, 9)
    mask = random_mask(1, vocab, g, 3).expand(rows, -1)[:, 1:]
    args = (x, tokens, None, None, rep, None, None, ids, values, mask)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.logits_process(*args)
    side.synchronize()
    check_logits(got, x, tokens, None, None, rep, None, None, ids, values, mask[:, :-(-vocab // 32)])
    # the same row by row
    for r in range(rows):
        one = ops.logits_process(*(None if t is None else t[r:r + 1] for t in args))
        assert torch.equal(one[0], got[r])


def test_logits_edges_of_rows(cuda_device, ops):
    """Rows of every length around the vectors' and pieces', each starting at
    another offset, logits and outputs aligned alike and not."""
    g = gen(25)
    pool = torch.randn(1 << 16, generator=g, device="cuda")
    for vocab in (*range(1, 12), 1021, 1022, 1023, 1024, 1025, 1026, 2047, 2050, 4099):
        for pad in range(4):
            rows, ld = 5, vocab + pad
            x = pool[pad:pad + rows * ld].view(rows, ld)[:, :vocab]
            mask = random_mask(rows, vocab, g)
            for dtype in (F32, BF16):
                y = x if dtype is F32 else pool.to(dtype)[pad:pad + rows * ld].view(rows, ld)[:, :vocab]
                tokens = torch.randint(0, vocab, (rows, 3), generator=g, device="cuda")
                freq = torch.ones(rows, device="cuda")
                got = ops.logits_process(y, tokens, frequency=freq, mask=mask)
                check_logits(got, y, tokens, None, None, None, freq, None, None, None, mask)


def test_logits_in_place_through_the_c_abi(cuda_device):
    import ctypes

    import cuda_transformer_b200 as cb
    g = gen(24)
    x = torch.randn(2, 5000, generator=g, device="cuda")
    tokens = torch.randint(0, 5000, (2, 90), generator=g, device="cuda")
    freq = torch.full((2,), 0.7, device="cuda")
    want, bound = logits_reference(x, tokens, None, None, None, freq, None, None, None, None)
    p = ctypes.c_void_p
    cb.check(cb.lib().ct_logits_process(
        p(x.data_ptr()), 5000, cb.DTYPE_F32, p(x.data_ptr()), 5000, 2, 5000, p(tokens.data_ptr()),
        90, 90, None, None, None, p(freq.data_ptr()), None, None, 0, None, 0, 0, None, 0,
        H._stream()))
    assert bool(((x.double() - want).abs() <= bound).all())


# ---------------------------------------------------------------- refusals
def test_refusals(cuda_device, ops):
    k = torch.zeros(4, 2, 8, 64, device="cuda")
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(3, 4, 64, device="cuda")
    ws = ops.paged_attention_workspace(4, 2, 64)

    def att(q=q, k=k, v=k, table=table, lens=lens, **kw):
        return ops.paged_attention(q, k, v, table, lens, **kw)

    att()
    for bad in (dict(q=q[:2]), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.double()),
                dict(q=q.to(BF16)), dict(v=k[:3]), dict(v=k.to(BF16)), dict(table=table.long()),
                dict(table=table[0]), dict(lens=lens.long()), dict(lens=lens[:2]),
                dict(lens=lens.cpu()), dict(k=k.transpose(2, 3), v=k.transpose(2, 3)),
                dict(workspace=ws[1:]), dict(workspace=ws[:16]), dict(workspace=ws.view(torch.int32)),
                dict(q=q[..., :48].contiguous(), k=k[..., :48].contiguous(),
                     v=k[..., :48].contiguous()),
                dict(k=torch.zeros(4, 2, 8, 65, device="cuda")[..., 1:],
                     v=torch.zeros(4, 2, 8, 65, device="cuda")[..., 1:])):
        with pytest.raises(RuntimeError):
            att(**bad)

    kn = torch.zeros(3, 2, 64, device="cuda")
    cos, sin = ops.rotary_tables(16, 64, device="cuda")

    def app(k_cache=k, v_cache=k.clone(), k=kn, v=kn, table=table, pos=lens, **kw):
        return ops.kv_append_(k_cache, v_cache, k, v, table, pos, **kw)

    app()
    for bad in (dict(k=kn[:2]), dict(k=kn[:, :1], v=kn[:, :1]), dict(k=kn.to(BF16), v=kn.to(BF16)),
                dict(pos=lens.long()), dict(pos=lens[:2]), dict(seq_ids=lens.long()), dict(cos=cos),
                dict(cos=cos, sin=sin[:8]), dict(cos=cos.double(), sin=sin.double()),
                dict(cos=torch.zeros(16, 33, device="cuda"), sin=torch.zeros(16, 33, device="cuda")),
                dict(q=kn[:2]), dict(q=kn.to(BF16)), dict(v=kn.to(BF16)), dict(table=table.float())):
        with pytest.raises(RuntimeError):
            app(**bad)

    x = torch.zeros(3, 100, device="cuda")
    tokens = torch.zeros(3, 5, dtype=torch.int64, device="cuda")
    one = torch.ones(3, device="cuda")
    for bad in (dict(tokens=tokens.int()), dict(tokens=tokens[:2]), dict(tokens=tokens, lens=lens.long()),
                dict(tokens=tokens, repetition=one[:2]), dict(tokens=tokens, frequency=one.double()),
                dict(bias_ids=tokens), dict(bias_ids=tokens, bias_values=one[:, None]),
                dict(mask=torch.zeros(3, 3, dtype=torch.int32, device="cuda")),
                dict(mask=torch.zeros(3, 4, dtype=torch.int64, device="cuda")),
                dict(tokens=tokens.cpu())):
        with pytest.raises(RuntimeError):
            ops.logits_process(x, **bad)
    with pytest.raises(RuntimeError):
        ops.logits_process(x.double())
    with pytest.raises(RuntimeError):
        ops.logits_process(x[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,hist", [(3, 5000, 4000), (2, 60000, 40000)])
def test_logits_penalty_is_a_division(cuda_device, ops, dtype, rows, vocab, hist):
    """x / r and x * r, each rounded once: the same bits as torch's.  (The longer histories
    exceed the list of tokens, so that both places that mend are met.)"""
    g = gen(vocab)
    x = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    tokens = torch.randint(0, vocab, (rows, hist), generator=g, device="cuda")
    rep = 1.0 + torch.rand(rows, generator=g, device="cuda")
    rep[0] = 1e-39                       # its reciprocal is beyond FP32
    seen = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, tokens, True)
    r, y = rep[:, None], x.float()
    want = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
    assert torch.equal(ops.logits_process(x, tokens, repetition=rep), want)


# ------------------------------------------------------- non-finite cached values
GROUPS = [(F32, F32, 1), (F32, F32, 2), (F32, F32, 5), (F32, BF16, 1), (F32, BF16, 2),
          (F32, BF16, 8), (F32, F16, 1), (F32, F16, 2), (F32, F16, 3), (BF16, BF16, 1),
          (BF16, BF16, 4), (F16, F16, 1), (F16, F16, 8), (F32, F32, 20), (BF16, BF16, 12)]


def infinite_case(act, cache, group, dim, seed):
    """Two key/value heads, sequences of one tile, of several and of several CTAs'
    shares; q is positive in dim 3, so that an infinite key there decides the sign."""
    lens, page, g = [9, 100, 3000], 16, gen(seed)
    k, v, table = make_cache(lens, 2, dim, page, cache, "token", g)
    q = torch.randn(3, 2 * group, dim, generator=g, device="cuda")
    q[:, :, 3] = q[:, :, 3].abs() + 0.1
    return lens, page, k, v, table, q.to(act)


def slot(table, b, j, page=16):
    return int(table[b, j // page]), slice(None), j % page


@pytest.mark.parametrize("act,cache,group", GROUPS)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_infinite_keys(cuda_device, ops, act, cache, group, dim):
    """A key whose score is -inf has no weight, wherever it lies; one whose score is +inf
    leaves no number."""
    lens, page, k, v, table, q = infinite_case(act, cache, group, dim, 40 + dim + group)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean_k, keep = k.clone(), [torch.ones(m, dtype=torch.bool) for m in lens]
    for b, m in enumerate(lens):
        for j in (0, m // 2, m - 1):
            k[slot(table, b, j)][..., 3] = -math.inf
            keep[b][j] = False
    got = ops.paged_attention(q, k, v, table, n)
    # the same without those keys
    k2, v2, table2 = make_cache([int(x.sum()) for x in keep], 2, dim, page, cache, "head", gen(1))
    for b, x in enumerate(keep):
        for i, j in enumerate(x.nonzero()[:, 0].tolist()):
            for new, old in ((k2, clean_k), (v2, v)):
                new[slot(table2, b, i)] = old[slot(table, b, j)]
    check_attention(q, k2, v2, table2, [int(x.sum()) for x in keep], page, got, dim ** -0.5)
    k[slot(table, 1, 50)][..., 3] = math.inf
    out, lse = ops.paged_attention(q, k, v, table, n)
    assert out[1].isnan().all()
    assert torch.equal(out[[0, 2]], got[0][[0, 2]]) and torch.equal(lse[[0, 2]], got[1][[0, 2]])


@pytest.mark.parametrize("act,cache,group", GROUPS)
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attention_infinite_values(cuda_device, ops, act, cache, group, dim):
    """An infinite value with a weight makes its dim of the result infinite, two of opposite
    signs NaN; the other dims are untouched.  Scores are kept within a few units, so that
    every weight is a normal number of each type."""
    lens, page, k, v, table, q = infinite_case(act, cache, group, dim, 80 + dim + group)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    clean = v.clone()
    want = ops.paged_attention(q, k, v, table, n)
    for b, m in enumerate(lens):
        v[slot(table, b, 0)][..., 5] = math.inf
        v[slot(table, b, m - 1)][..., dim - 2] = -math.inf
        v[slot(table, b, m // 2)][..., dim // 2] = math.inf
        v[slot(table, b, m // 3)][..., dim // 2] = -math.inf
    out, lse = ops.paged_attention(q, k, v, table, n)
    assert torch.equal(lse, want[1])
    assert (out[..., 5] == math.inf).all() and (out[..., dim - 2] == -math.inf).all()
    assert out[..., dim // 2].isnan().all()
    rest = [d for d in range(dim) if d not in (5, dim - 2, dim // 2)]
    assert torch.equal(out[..., rest], want[0][..., rest])
    check_attention(q, k, clean, table, lens, page, want, dim ** -0.5)


# ---------------------------------------------------------------- forms seldom met
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("heads,kv,dim", [(3, 3, 64), (4, 2, 32), (5, 1, 128), (12, 1, 64),
                                          (16, 2, 64)])
def test_attention_query_layouts(cuda_device, ops, act, cache, heads, kv, dim):
    """q that is not made of 16-byte vectors (a last stride other than one, an odd offset, an odd
    row stride) is read element by element: the same bits as its dense copy."""
    lens, g = [40, 0, 700, 3], gen(heads + dim)
    k, v, table = make_cache(lens, kv, dim, 16, cache, "token", g)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    flat = torch.randn(4 * (heads + 1) * (2 * dim + 3) + 5, generator=g, device="cuda").to(act)
    views = (torch.as_strided(flat, (4, heads, dim), (heads * 2 * dim, 2 * dim, 2), 1),
             torch.as_strided(flat, (4, heads, dim), (heads * dim, dim, 1), 1),
             torch.as_strided(flat, (4, heads, dim), (heads * (dim + 3), dim + 3, 1), 0),
             torch.as_strided(flat, (4, heads, dim), (heads * dim, 1, heads), 0),
             torch.as_strided(flat, (4, heads, dim), (0, dim, 1), 3))
    for q in views:
        got = ops.paged_attention(q, k, v, table, n)
        want = ops.paged_attention(q.contiguous(), k, v, table, n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        check_attention(q, k, v, table, lens, 16, got, dim ** -0.5)


# rows of 128 parts that a token's heads make (FP32: four elements a part's vector, 16-bit: eight,
# or one), and the parts a thread that follow: 2, 3, 4, 3 with a partly filled block of y
@pytest.mark.parametrize("act,cache,heads,kv,dim,rot,interleaved,vec,rows", [
    (F32, BF16, 16, 8, 64, 64, False, 4, 2), (F32, F32, 32, 8, 64, 32, True, 4, 3),
    (F32, F16, 48, 8, 64, 64, False, 4, 4), (F32, BF16, 50, 10, 64, 64, False, 4, 5),
    (BF16, BF16, 100, 6, 128, 128, False, 8, 7), (F16, F16, 28, 2, 128, 64, True, 8, 2),
    (F32, F16, 32, 4, 32, 6, False, 1, 5), (F16, F16, 12, 2, 32, 10, True, 1, 2),
    (BF16, BF16, 18, 3, 64, 2, False, 1, 6), (F32, F32, 40, 12, 32, 2, True, 1, 8)])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_append_many_tokens(cuda_device, ops, act, cache, heads, kv, dim, rot, interleaved, vec,
                            rows, layout):
    """Prompts long enough that a thread has several parts of a token's heads."""
    assert -(-(heads + 2 * kv) * (dim // (2 * vec)) // 128) == rows
    sms, page, g = torch.cuda.get_device_properties(0).multi_processor_count, 13, gen(rows + dim)
    tokens = -(-128 * sms // rows) + 5
    lens = [tokens // 3, tokens - tokens // 3]
    need = [-(-n // page) for n in lens]
    table = torch.full((2, max(need)), -1, dtype=torch.int32, device="cuda")
    perm = torch.randperm(sum(need) + 2, generator=g, device="cuda").int()
    table[0, :need[0]], table[1, :need[1]] = perm[:need[0]], perm[need[0]:sum(need)]
    shape = (sum(need) + 2, kv, page, dim)
    if layout == "token":
        shape = (shape[0], page, kv, dim)
    k_cache, v_cache = (torch.full(shape, 7.0, dtype=cache, device="cuda") for _ in range(2))
    if layout == "token":
        k_cache, v_cache = k_cache.transpose(1, 2), v_cache.transpose(1, 2)
    ids = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)]).int().cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    pos[5], pos[tokens - 2] = -1, -1           # padding
    there = pos >= 0
    qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=g, device="cuda").to(act)
    q, k, v = qkv.split([heads, kv, kv], 1)
    cos, sin = ops.rotary_tables(max(lens), rot, device="cuda")
    want_k, want_v = k_cache.double(), v_cache.clone()
    q_out, k_out = ops.kv_append_(k_cache, v_cache, k, v, table, pos, seq_ids=ids, q=q, cos=cos,
                                  sin=sin, interleaved=interleaved, want_k=True)
    assert torch.count_nonzero(q_out[~there]) == torch.count_nonzero(k_out[~there]) == 0
    ids, pos, qd, kd, vd = (t[there] for t in (ids, pos, q, k, v))
    qr, qb = rotate(qd, pos, cos, sin, interleaved)
    kr, kb = rotate(kd, pos, cos, sin, interleaved)
    for got, ref, bound in ((q_out[there], qr, qb), (k_out[there], kr, kb)):
        assert bool(((got.double() - ref).abs() <= bound + ROUND[act] * ref.abs() + 2.0 ** -25).all())
    where = (table[ids.long(), pos.long() // page].long(), slice(None), pos.long() % page)
    want_k[where], want_v[where] = kr, vd.to(cache)
    bound = torch.zeros_like(want_k)
    bound[where] = kb + ROUND[cache] * kr.abs() + 2.0 ** -25
    assert bool(((k_cache.double() - want_k).abs() <= bound).all())
    assert torch.equal(v_cache, want_v)


def test_operators_keep_their_schemas(cuda_device, ops):
    """Outputs are tensors of their own, only what the schema names is written, and the fake
    kernels give the shapes and types of the real ones."""
    g = gen(31)
    k, v = (torch.randn(4, 2, 8, 64, generator=g, device="cuda") for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3], [1, 0]], dtype=torch.int32, device="cuda")
    n = torch.tensor([3, 9, 0], dtype=torch.int32, device="cuda")
    q, kn = (torch.randn(3, h, 64, generator=g, device="cuda") for h in (4, 2))
    cos, sin = ops.rotary_tables(16, 64, device="cuda")
    x = torch.randn(3, 50, generator=g, device="cuda").half()
    tokens = torch.randint(0, 50, (3, 7), generator=g, device="cuda")
    ct = torch.ops.cuda_transformer
    ws = ops.paged_attention_workspace(4, 2, 64)
    for op, args in ((ct.kv_append_, (k, v, kn, kn, table, n, None, None, None, None, False, False)),
                     (ct.kv_append_, (k, v, kn, kn, table, n, None, q, cos, sin, False, True)),
                     (ct.paged_attention, (q, k, v, table, n, 0.125, ws)),
                     (ct.paged_attention, (q, k, v, table, n, 0.125, None)),
                     (ct.logits_process, (x, tokens, n, None, None, None, None, None, None, None))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))
    a, b = ops.kv_append_(k, v, kn, kn, table, n)
    assert a is not b


@pytest.mark.parametrize("rows", [1, 200])
def test_logits_biases_of_a_whole_vocabulary(cuda_device, ops, rows):
    """Tens of thousands of entries a row, in any order, tokens listed twice far apart and one
    listed hundreds of times.  The result does not depend on the number of rows (by which a
    block's part of a row is chosen): entries are added one by one in their order."""
    g = gen(91)
    vocab = 20011
    x = torch.randn(1, vocab, generator=g, device="cuda")
    ids = torch.cat([torch.randperm(vocab, generator=g, device="cuda"),
                     torch.full((700,), 5, device="cuda"),
                     torch.randint(-3, vocab + 3, (vocab,), generator=g, device="cuda")])[None]
    values = torch.randn(ids.shape, generator=g, device="cuda")
    got = ops.logits_process(x.expand(rows, -1), bias_ids=ids.expand(rows, -1),
                             bias_values=values.expand(rows, -1))
    ok = (ids[0] >= 0) & (ids[0] < vocab)
    at, w = ids[0][ok], values[0][ok]
    add = lambda t: torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, t)  # noqa: E731
    ref = x[0].double() + add(w.double())
    # a rounding of 2^-24 for each entry, of sums no larger than this
    bound = 2.0 ** -24 * add(torch.ones_like(w).double()) * (x[0].abs() + add(w.abs().double()))
    assert bool(((got.double() - ref).abs() <= bound).all())
    total = x[0].cpu().numpy().copy()
    for i, v in zip(at.tolist(), w.cpu().numpy()):
        total[i] += v
    assert torch.equal(got, torch.from_numpy(total).cuda().expand(rows, -1))


def test_logits_time_of_many_biases(cuda_device, ops):
    """100256 entries take a few thousand times as long as none at most, not the square of it:
    well below a fifth of a second (a scan of all entries for each took 1.8 s)."""
    vocab = 100256
    x, values = (torch.zeros(1, vocab, device="cuda") for _ in range(2))
    ids = torch.arange(vocab, device="cuda")[None]
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(2):
        start.record()
        ops.logits_process(x, bias_ids=ids, bias_values=values)
        end.record()
    torch.cuda.synchronize()
    assert start.elapsed_time(end) < 200.0


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_sums_of_long_sequences(cuda_device, ops, dim):
    """Half a million keys in one block's hands (as many sequences as that takes, on the same
    pages), values about 1: sums that were cut off a little at each of some 8000 steps a warp
    would be short by 2^-10.  f16 rounds by 2^-11 of the result at most; 8192 roundings of
    2^-24 that point either way add 2^-17.5, of which 2^-15 is a sixfold."""
    n, page, g = 1 << 19, 128, gen(dim)
    batch = 3 * torch.cuda.get_device_properties(0).multi_processor_count + 6
    k = (0.05 * torch.randn(n // page, 1, page, dim, generator=g, device="cuda")).to(F16)
    v = (1 + 0.01 * torch.randn(k.shape, generator=g, device="cuda")).to(F16)
    table = torch.arange(n // page, device="cuda").int().expand(batch, -1)
    q = torch.randn(batch, 8, dim, generator=g, device="cuda").to(F16)
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out, _ = ops.paged_attention(q, k, v, table, lens)
    kk, vv = (t[:, 0].flatten(0, 1).double() for t in (k, v))
    for b in (0, batch // 2, batch - 1):
        ref = (q[b].double() @ kk.T * dim ** -0.5).softmax(-1) @ vv
        assert bool(((out[b].double() - ref).abs() <= (2.0 ** -11 + 2.0 ** -15) * ref.abs()).all())


def test_strides_of_single_elements(cuda_device, ops):
    """One page, one key/value head, slots of one, one token, one sequence: their strides say
    nothing, and the results are those of dense tensors."""
    g = gen(61)
    lens = torch.tensor([9], dtype=torch.int32, device="cuda")
    cos, sin = ops.rotary_tables(16, 64, device="cuda")
    for pages, kv, page in ((1, 1, 16), (16, 1, 1), (1, 2, 16)):
        for cache in (F32, BF16):
            k, v = (torch.randn(pages, kv, page, 64, generator=g, device="cuda").to(cache)
                    for _ in range(2))
            table = torch.arange(16 if page == 1 else 1, device="cuda").int()[None]
            q = torch.randn(1, 4 * kv, 64, generator=g, device="cuda")
            kn, vn = (torch.randn(1, kv, 64, generator=g, device="cuda") for _ in range(2))

            def odd(t):
                s = [3 + 2 * i if n == 1 else st for i, (n, st) in enumerate(zip(t.shape, t.stride()))]
                return torch.as_strided(t, t.shape, s)

            want = ops.paged_attention(q, k, v, table, lens)
            got = ops.paged_attention(odd(q), odd(k), odd(v), table, lens)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            k2, v2 = k.clone(), v.clone()
            a = ops.kv_append_(k, v, kn, vn, table, lens, q=q, cos=cos, sin=sin, want_k=True)
            b = ops.kv_append_(odd(k2), odd(v2), odd(kn), odd(vn), table, lens, q=odd(q), cos=cos,
                               sin=sin, want_k=True)
            assert all(torch.equal(x, y) for x, y in zip((*a, k, v), (*b, k2, v2)))
    q_out, k_out = ops.kv_append_(k, v, kn, vn, torch.zeros(0, 3, dtype=torch.int32, device="cuda"),
                                  lens, want_k=True)
    assert k_out.isnan().all()
