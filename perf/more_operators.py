"""Measured cases of the speculative-decoding operators.

A drafter proposes several tokens after a sequence's last one, as a chain or as
a tree; the model looks at all of them in one step.  Four operators of such a
step: ``tree_attention`` (the drafted tokens against the paged cache, each with
the cached tokens and its own ancestors), ``verify_drafts`` (which of them are
kept, by the target's and the drafter's probabilities and given random numbers,
and the token after them), ``kv_compact_`` (the kept tokens' keys and values
move up to where a plain sequence has them) and ``kv_copy_pages_`` (pages of a
sequence that is forked).

``run`` computes a case either with the framework's kernels (``own``) or in
plain torch operations; ``exact`` computes it in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------- cases
def attention(name, batch, drafts, tree, ragged, q_heads, kv_heads, dim, low, high, page, act,
              cache, layout):
    """`drafts` tokens a sequence (`ragged`: up to so many), a tree or a chain;
    `low`..`high`: range of the cached lengths before them."""
    return {"name": name, "op": "attention", "batch": batch, "drafts": drafts, "tree": tree,
            "ragged": ragged, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "low": low,
            "high": high, "page": page, "act": act, "cache": cache, "layout": layout}


def verify(name, batch, drafts, tree, ragged, vocab, mode, near, act):
    """`mode`: "sample" (tokens drawn from a drafter's probabilities), "lookup"
    (certain proposals, the target's probabilities) or "greedy" (the best
    token of the target's scores); `near`: how close the drafter is."""
    return {"name": name, "op": "verify", "batch": batch, "drafts": drafts, "tree": tree,
            "ragged": ragged, "vocab": vocab, "mode": mode, "near": near, "act": act}


def compact(name, batch, low, high, drafts, kept, layers, kv_heads, dim, page, cache, layout):
    """`kept` (a share) of the `drafts` tokens after the first `low`..`high` stay."""
    return {"name": name, "op": "compact", "batch": batch, "low": low, "high": high,
            "drafts": drafts, "kept": kept, "layers": layers, "kv_heads": kv_heads, "dim": dim,
            "page": page, "cache": cache, "layout": layout}


def copy(name, count, layers, kv_heads, dim, page, cache, layout):
    """`count` pages of every layer's keys and values."""
    return {"name": name, "op": "copy", "count": count, "layers": layers, "kv_heads": kv_heads,
            "dim": dim, "page": page, "cache": cache, "layout": layout}


def listed():
    return [
        # the character GPT (6 heads of 64, context 256) with a small tree: latency
        attention("tree_char_gpt", 8, 8, True, False, 6, 6, 64, 1, 248, 16, "f32", "f32", "head"),
        # a busy server: trees of 16 over conversations of very different lengths
        attention("tree_serve_bf16", 64, 16, True, False, 32, 8, 128, 16, 4096, 16, "bf16",
                  "bf16", "token"),
        # one long document and a large tree: many rows for each key
        attention("tree_long_bf16", 1, 64, True, False, 32, 8, 128, 131072, 131072, 64, "bf16",
                  "bf16", "token"),
        # the FP32 model's heads over a half-width cache, chains of up to 5
        attention("chain_f32_bf16cache", 16, 5, False, True, 32, 32, 64, 3500, 4096, 32, "f32",
                  "bf16", "head"),
        # all query heads on one key/value head, f16, odd sizes of trees and pages
        attention("tree_mqa_f16", 32, 33, True, True, 16, 1, 64, 1, 16384, 24, "f16", "f16",
                  "token"),
        # one answer with a draft model, 7 tokens ahead: latency
        verify("verify_one", 1, 8, False, False, 100256, "sample", 0.5, "f32"),
        # a server's step: trees of 16, several candidates at a place
        verify("verify_serve", 64, 16, True, False, 100256, "sample", 0.7, "f32"),
        # proposals looked up in the text, best tokens only, an odd vocabulary
        verify("verify_greedy", 128, 8, False, True, 50257, "greedy", 0.6, "f32"),
        # the kept path of each of 64 trees, in 12 layers
        compact("compact_trees", 64, 16, 2048, 16, 0.25, 12, 8, 128, 16, "bf16", "token"),
        # half of long sequences dropped (tokens that no head looks at)
        compact("compact_long", 4, 1, 1, 8192, 0.5, 4, 32, 64, 32, "bf16", "head"),
        # the last pages of a few forked sequences: latency
        copy("copy_few", 8, 6, 6, 64, 16, "f32", "head"),
        # a pool's worth of pages, 12 layers
        copy("copy_many", 512, 12, 8, 128, 16, "bf16", "token"),
    ]


def spread(rng, low, high):
    """A whole number of low..high, uniform over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "verify", "verify", "compact", "copy"])
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                             ("f16", "f16")])
    layout, page = rng.choice(["head", "token"]), rng.choice([1, 8, 13, 16, 24, 32, 64, 128])
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
    tree, ragged = rng.random() < 0.6, rng.random() < 0.4
    if op == "attention":
        q_heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if g * kv_heads <= 64])
        drafts = spread(rng, 1, 128)
        # at most 2**28 bytes in each of K and V and 2**28 scores, as the largest listed cases
        tokens = min(2 ** 28 // (kv_heads * dim * WIDTH[cache]), 2 ** 28 // (q_heads * drafts),
                     2 ** 35 // (q_heads * drafts * dim))
        high = spread(rng, 1, max(1, min(131072, tokens) - drafts))
        batch = spread(rng, 1, max(1, min(256, tokens // (high + drafts))))
        c = attention("", batch, drafts, tree, ragged, q_heads, kv_heads, dim,
                      spread(rng, 1, high), high, page, act, cache, layout)
    elif op == "verify":
        vocab = spread(rng, 65, 200000)
        drafts = spread(rng, 2, 64)
        batch = spread(rng, 1, max(1, min(256, 100000000 // (vocab * drafts))))
        c = verify("", batch, drafts, tree, ragged, vocab,
                   rng.choice(["sample", "sample", "lookup", "greedy"]), rng.uniform(0.3, 0.9),
                   rng.choice(["f32", "f32", "bf16", "f16"]))
    elif op == "compact":
        layers = rng.randint(1, 16)
        # at most 2**30 bytes of caches
        tokens = 2 ** 30 // (2 * layers * kv_heads * dim * WIDTH[cache])
        drafts = spread(rng, 2, max(2, min(tokens // 8, 8192)))
        high = spread(rng, 1, max(1, min(2048, tokens // 4)))
        batch = spread(rng, 1, max(1, min(256, tokens // (high + drafts + page))))
        c = compact("", batch, spread(rng, 1, high), high, drafts, rng.uniform(0.1, 0.9), layers,
                    kv_heads, dim, page, cache, layout)
    else:
        layers = rng.randint(1, 16)
        count = spread(rng, 1, max(1, min(4096, 2 ** 29 // (2 * layers * kv_heads * dim * page
                                                             * WIDTH[cache]))))
        c = copy("", count, layers, kv_heads, dim, page, cache, layout)
    c.pop("name")
    return c


def lengths(case):
    """The case's lengths, the same for every seed: low..high, evenly over the logarithm."""
    low, high, count = case["low"], case["high"], case["batch"]
    if count == 1:
        return [high]
    return [min(high, max(low, round(low * (high / low) ** (i / (count - 1)))))
            for i in range(count)]


def draft_counts(case):
    """Drafted tokens (verify: the last token too) of each sequence, the same for every seed."""
    n = case["drafts"]
    return [1 + (7 * i) % n if case["ragged"] else n for i in range(case["batch"])]


# ------------------------------------------------------------------ inputs
def page_table(lens, page, gen, device):
    """Pages for sequences of `lens` tokens, scattered over a pool a little larger
    than needed; entries past a sequence's end are 0."""
    need = torch.tensor([max(1, -(-n // page)) for n in lens])
    total, width = int(need.sum()), int(need.max())
    pool = total + total // 8 + 1
    perm = torch.randperm(pool, generator=gen, device=device)[:total].int()
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=device)
    filled = (torch.arange(width)[None, :] < need[:, None]).to(device)
    table[filled] = perm
    return table, pool


def cache_tensors(case, pool, count, gen, device):
    """Caches, indexed [page, head, slot, dim]; "token" keeps the heads of one
    token together in memory, "head" the slots of one head."""
    h, s, d, kind = case["kv_heads"], case["page"], case["dim"], DTYPES[case["cache"]]
    shape = (pool, s, h, d) if case["layout"] == "token" else (pool, h, s, d)
    tensors = [torch.randn(shape, generator=gen, device=device, dtype=kind) for _ in range(count)]
    return [t.transpose(1, 2) if case["layout"] == "token" else t for t in tensors]


def draft_parents(case, gen, device):
    """int32 [batch, drafts]: in a tree a node follows one of the four before it,
    in a chain the one before it; -1: none."""
    batch, n = case["batch"], case["drafts"]
    at = torch.arange(n, device=device)
    back = (torch.randint(0, 4, (batch, n), generator=gen, device=device) if case["tree"]
            else torch.zeros(batch, n, dtype=torch.int64, device=device))
    return torch.where(at > 0, (at - 1 - back).clamp(min=0), -1).int()


def ancestors(parents):
    """bool [batch, drafts, drafts]: which drafted tokens each one sees."""
    batch, n = parents.shape
    sees = torch.eye(n, dtype=torch.bool, device=parents.device).repeat(batch, 1, 1)
    rows = torch.arange(batch, device=parents.device)
    for i in range(1, n):
        sees[:, i] |= sees[rows, parents[:, i].long()]
    return sees


def packed(bits):
    """bool [..., n] as int32 [..., ceil(n / 32)]."""
    words = -(-bits.shape[-1] // 32)
    wide = torch.nn.functional.pad(bits, (0, 32 * words - bits.shape[-1])).unflatten(-1, (words, 32))
    value = (wide.long() << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(value >= 2 ** 31, value - 2 ** 32, value).int()


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    order = random.Random(seed)
    state = {"case": case}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    if case["op"] == "attention":
        lens = list(zip(lengths(case), draft_counts(case)))
        order.shuffle(lens)
        table, pool = page_table([a + b for a, b in lens], case["page"], gen, device)
        state["k_cache"], state["v_cache"] = cache_tensors(case, pool, 2, gen, device)
        state["table"] = table
        state["context_lens"], state["draft_lens"] = ints([a for a, _ in lens]), None
        if case["ragged"]:
            state["draft_lens"] = ints([b for _, b in lens])
        state["mask"] = None
        if case["tree"]:
            state["mask"] = packed(ancestors(draft_parents(case, gen, device)))
        # q is a view of a fused projection, as the GPT's blocks make it
        h = case["q_heads"] + 2 * case["kv_heads"]
        qkv = torch.randn(case["batch"], case["drafts"], h, case["dim"], generator=gen,
                          device=device).to(DTYPES[case["act"]])
        state["q"] = qkv[:, :, :case["q_heads"]]
    elif case["op"] == "verify":
        batch, n, vocab, kind = case["batch"], case["drafts"], case["vocab"], DTYPES[case["act"]]
        counts = draft_counts(case)
        order.shuffle(counts)
        state["draft_lens"] = ints(counts) if case["ragged"] else None
        state["parents"] = draft_parents(case, gen, device) if case["tree"] else None
        before = draft_parents(dict(case), gen, device).long().clamp(min=0)
        if case["tree"]:
            before = state["parents"].long().clamp(min=0)
        # logits of a trained model are a few units wide; the drafter's are near them
        logits = 3.0 * torch.randn(batch, n, vocab, generator=gen, device=device)
        rows = torch.arange(batch, device=device)[:, None]
        state["draft_probs"] = state["uniform"] = None
        far = 3.0 * (1.0 - case["near"]) / case["near"] if case["mode"] == "sample" else 0.0
        drafter = torch.softmax(logits + far * torch.randn(logits.shape, generator=gen,
                                                           device=device), -1)
        tokens = torch.multinomial(drafter[rows, before].flatten(0, 1), 1, generator=gen)
        tokens = tokens.view(batch, n)
        if case["mode"] != "sample":  # proposals hit the target's best token now and then
            hit = torch.rand(batch, n, generator=gen, device=device) < case["near"]
            tokens = torch.where(hit, logits.argmax(-1).gather(1, before), tokens)
        state["tokens"] = tokens
        if case["mode"] == "greedy":
            state["target"] = logits.to(kind)
        else:
            state["target"] = torch.softmax(logits, -1).to(kind)
            state["uniform"] = torch.rand(batch, n, generator=gen, device=device)
            if case["mode"] == "sample":
                state["draft_probs"] = drafter.to(kind)
    elif case["op"] == "compact":
        lens, n = lengths(case), case["drafts"]
        order.shuffle(lens)
        table, pool = page_table([a + n for a in lens], case["page"], gen, device)
        state["caches"] = cache_tensors(case, pool, 2 * case["layers"], gen, device)
        state["table"], state["context_lens"] = table, ints(lens)
        # the first is always kept; the others come with the given share
        kept = torch.rand(case["batch"], n, generator=gen, device=device) < case["kept"]
        kept[:, 0] = True
        state["counts"] = kept.sum(1).int()
        at = torch.arange(n, device=device)
        keep = torch.where(kept, at, n).sort(1).values
        state["keep"] = torch.where(keep < n, keep, -1).int()
    else:
        n = case["count"]
        state["caches"] = cache_tensors(case, 2 * n + 3, 2 * case["layers"], gen, device)
        pages = torch.randperm(2 * n + 3, generator=gen, device=device).int()
        state["src"], state["dst"] = pages[:n], pages[n:2 * n]
    return state


# -------------------------------------------------------------------- runs
def run(state):
    return (run_own if own else run_plain)[state["case"]["op"]](state)


def own_attention(s):
    from cuda_transformer import ops

    return ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["context_lens"],
                              draft_lens=s["draft_lens"], mask=s["mask"])


def own_verify(s):
    from cuda_transformer import ops

    return ops.verify_drafts(s["target"], s["tokens"], parents=s["parents"],
                             draft_lens=s["draft_lens"], draft_probs=s["draft_probs"],
                             uniform=s["uniform"])


def own_compact(s):
    from cuda_transformer import ops

    ops.kv_compact_(s["caches"], s["table"], s["context_lens"], s["keep"], s["counts"])
    return s["caches"]


def own_copy(s):
    from cuda_transformer import ops

    ops.kv_copy_pages_(s["caches"], s["src"], s["dst"])
    return s["caches"]


def visible(s, places):
    """bool [batch, drafts, places]: which cached positions each drafted token sees."""
    batch, n, device = s["case"]["batch"], s["case"]["drafts"], s["table"].device
    at, ids = torch.arange(places, device=device), torch.arange(n, device=device)
    context = s["context_lens"][:, None]
    lens = n if s["draft_lens"] is None else s["draft_lens"][:, None]
    if s["mask"] is None:
        sees = (ids[:, None] >= ids).expand(batch, n, n)
    else:
        sees = (s["mask"][:, :, ids // 32] >> (ids % 32)) & 1 != 0
    index = (at - context).clamp(0, n - 1)[:, None].expand(batch, n, places)
    drafted = ((at >= context) & (at < context + lens))[:, None]
    there = (at < context)[:, None] | (drafted & sees.gather(2, index))
    return there & (ids < lens)[..., None]


def plain_attention(s):
    q, table = s["q"].float(), s["table"].long()
    batch, n, heads, dim = q.shape
    kv = s["k_cache"].shape[1]
    group = heads // kv
    k, v = (c[table].float().transpose(1, 2).reshape(batch, kv, -1, dim)
            for c in (s["k_cache"], s["v_cache"]))
    rows = q.reshape(batch, n, kv, group, dim).transpose(1, 2).reshape(batch, kv, n * group, dim)
    scores = rows @ k.transpose(2, 3) * dim ** -0.5
    there = visible(s, k.shape[2])[:, None, :, None]
    scores = torch.where(there, scores.unflatten(2, (n, group)), -math.inf).flatten(2, 3)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    out, lse = (x.unflatten(2, (n, group)).transpose(1, 2).reshape(batch, n, heads, -1)
                for x in (out, lse))
    return out.to(s["q"].dtype), lse[..., 0]


def plain_verify(s):
    """A node is looked at once, in order: its parent, when that is the last one
    kept, has had its earlier children refused.  What is compared and summed is
    held in 64 bits."""
    target, tokens = s["target"], s["tokens"]
    batch, n, vocab = target.shape
    device = target.device
    rows, ids = torch.arange(batch, device=device), torch.arange(vocab, device=device)
    lens = (torch.full((batch,), n, device=device) if s["draft_lens"] is None
            else s["draft_lens"].long())
    parents = (torch.arange(-1, n - 1, device=device).expand(batch, n) if s["parents"] is None
               else s["parents"].long())
    greedy = s["uniform"] is None
    current = torch.zeros(batch, dtype=torch.int64, device=device)
    kept = torch.zeros(batch, n, dtype=torch.bool, device=device)
    kept[:, 0] = lens > 0
    if greedy:
        top = target.float()
        best = torch.where(top == top.amax(-1, keepdim=True), ids, vocab).amin(-1)
    else:
        uniform = s["uniform"].double()
        rest, total = target[:, 0].double(), torch.ones(batch, dtype=torch.float64, device=device)
    for i in range(1, n):
        child = (parents[:, i] == current) & (i < lens)
        x = tokens[:, i]
        if greedy:
            yes = child & (x == best[rows, current])
        else:
            mass = rest[rows, x]
            if s["draft_probs"] is None:
                yes = child & (uniform[:, i] * total < mass)
                left, sum_left = torch.where(ids == x[:, None], 0.0, rest), total - mass
            else:
                drafter = s["draft_probs"][rows, current].double()
                yes = child & (uniform[:, i] * drafter[rows, x] * total < mass)
                left = (rest / total[:, None] - drafter).clamp_(min=0.0)
                sum_left = left.sum(-1)
            no = child & ~yes & (sum_left > 0)
            rest = torch.where(yes[:, None], target[:, i].double(),
                               torch.where(no[:, None], left, rest))
            total = torch.where(yes, 1.0, torch.where(no, sum_left, total))
        current = torch.where(yes, i, current)
        kept[:, i] = yes
    if greedy:
        last = best[rows, current]
    else:
        upto = rest.cumsum(-1)
        last = (upto <= (uniform[:, 0] * upto[:, -1])[:, None]).sum(-1).clamp(max=vocab - 1)
    counts = kept.sum(-1)
    at = torch.arange(n, device=device)
    path = torch.where(kept, at, n).sort(-1).values
    there = path < n
    new = tokens.gather(1, path.roll(-1, 1).clamp(max=n - 1))
    new = torch.where(at < counts[:, None] - 1, new, -1)
    new = torch.where((at == counts[:, None] - 1), last[:, None], new)
    return new, torch.where(there, path, -1).int(), counts.int()


def plain_compact(s):
    page = s["case"]["page"]
    at = torch.arange(s["keep"].shape[1], device=s["table"].device)
    there = at < s["counts"][:, None]
    # what is not kept repeats the first move
    keep = torch.where(there, s["keep"], s["keep"][:, :1].clamp(min=0)).long()
    base = s["context_lens"][:, None].long()
    rows = torch.arange(len(base), device=base.device)[:, None]
    src, dst = base + keep, base + torch.where(there, at, 0)
    from_page, to_page = (s["table"][rows, x // page].long() for x in (src, dst))
    for c in s["caches"]:
        c[to_page, :, dst % page] = c[from_page, :, src % page]
    return s["caches"]


def plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for c in s["caches"]:
        c[dst] = c[src]
    return s["caches"]


run_own = {"attention": own_attention, "verify": own_verify, "compact": own_compact,
           "copy": own_copy}
run_plain = {"attention": plain_attention, "verify": plain_verify, "compact": plain_compact,
             "copy": plain_copy}


# ------------------------------------------------------------------- exact
def exact_attention(s):
    q, page = s["q"].double(), s["case"]["page"]
    batch, n, heads, dim = q.shape
    group = heads // s["k_cache"].shape[1]
    out = torch.zeros_like(q)
    lse = torch.full((batch, n, heads), -math.inf, dtype=torch.float64, device=q.device)
    for b, context in enumerate(s["context_lens"].tolist()):
        m = n if s["draft_lens"] is None else int(s["draft_lens"][b])
        pages = s["table"][b, :-(-(context + m) // page)].long()
        k, v = (c[pages].permute(1, 0, 2, 3).flatten(1, 2)[:, :context + m].double()
                for c in (s["k_cache"], s["v_cache"]))
        if s["mask"] is None:
            sees = torch.ones(m, m, device=q.device).tril() > 0
        else:
            bits = (s["mask"][b, :m, :, None] >> torch.arange(32, device=q.device)) & 1
            sees = bits.flatten(1)[:, :m] > 0
        for h in range(heads):
            z = q[b, :m, h] @ k[h // group].T / math.sqrt(dim)
            z[:, context:] = z[:, context:].masked_fill(~sees, -math.inf)
            out[b, :m, h] = z.softmax(-1) @ v[h // group]
            lse[b, :m, h] = z.logsumexp(-1)
    return out, lse


def exact_verify(s):
    """From the root down, a place's candidates one after the other."""
    batch, n, vocab = s["target"].shape
    tokens, greedy = s["tokens"].tolist(), s["uniform"] is None
    parents = ([list(range(-1, n - 1))] * batch if s["parents"] is None else s["parents"].tolist())
    lens = [n] * batch if s["draft_lens"] is None else s["draft_lens"].tolist()
    new, paths = torch.full((batch, n), -1), torch.full((batch, n), -1)
    for b in range(batch):
        path, out = [], []
        node = 0 if lens[b] > 0 else None
        while node is not None:
            path.append(node)
            children = [i for i in range(node + 1, lens[b]) if parents[b][i] == node]
            p, node = s["target"][b, node].double(), None
            drafter = None if s["draft_probs"] is None else s["draft_probs"][b, path[-1]].double()
            if greedy:
                best = int((p == p.max()).nonzero()[0])
                node = next((i for i in children if tokens[b][i] == best), None)
            else:
                total = 1.0
                for i in children:
                    x, u = tokens[b][i], float(s["uniform"][b, i])
                    ask = u * total if drafter is None else u * total * float(drafter[x])
                    if ask < float(p[x]):
                        node = i
                        break
                    left = p.clone()
                    if drafter is None:
                        left[x] = 0.0
                        rest = total - float(p[x])
                    else:
                        left = torch.relu(p / total - drafter)
                        rest = float(left.sum())
                    if rest > 0:
                        p, total = left, rest
                if node is None:
                    upto = p.cumsum(0)
                    mark = (float(s["uniform"][b, 0]) * upto[-1]).reshape(1)
                    best = min(vocab - 1, int(torch.searchsorted(upto, mark, right=True)))
            out.append(best if node is None else tokens[b][node])
        new[b, :len(out)], paths[b, :len(path)] = torch.tensor(out), torch.tensor(path)
    return new.cuda(), paths.int().cuda(), (paths >= 0).sum(1).int().cuda()


def exact_compact(s):
    page, found = s["case"]["page"], [c.double() for c in s["caches"]]
    for b, base in enumerate(s["context_lens"].tolist()):
        keep = s["keep"][b, :int(s["counts"][b])].long()
        ends = []
        for at in (base + keep, base + torch.arange(len(keep), device=keep.device)):
            ends.append((s["table"][b, at // page].long(), at % page))
        for c in found:
            rows = c.transpose(1, 2)[ends[0]]
            c.transpose(1, 2)[ends[1]] = rows
    return found


def exact_copy(s):
    found = [c.double() for c in s["caches"]]
    for c in found:
        c.index_copy_(0, s["dst"].long(), c.index_select(0, s["src"].long()))
    return found


def exact(case, seed):
    calls = {"attention": exact_attention, "verify": exact_verify, "compact": exact_compact,
             "copy": exact_copy}
    return calls[case["op"]](prepare(case, seed))


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attention":
        lens = [(a, b) for a, b in zip(lengths(case), draft_counts(case))]
        row = case["kv_heads"] * case["dim"]
        rows = sum(b for _, b in lens) * case["q_heads"]
        moved = 2 * sum(a + b for a, b in lens) * row * WIDTH[case["cache"]]
        moved += 2 * rows * case["dim"] * WIDTH[case["act"]] + 4 * rows
        moved += 4 * sum(-(-(a + b) // case["page"]) for a, b in lens) + 8 * case["batch"]
        # context keys for each drafted token; drafted ones at half of a square
        seen = sum(b * a + b * (b + 1) // 2 for a, b in lens)
        return {"bytes": moved, "flops": 4 * case["q_heads"] * case["dim"] * seen}
    if case["op"] == "verify":
        # one row a sequence (two with a drafter): where the last token comes from
        rows = case["batch"] * (2 if case["mode"] == "sample" else 1)
        small = case["batch"] * case["drafts"] * (8 + 8 + 4 + 4 + 4)
        return {"bytes": rows * case["vocab"] * WIDTH[case["act"]] + small,
                "flops": 2 * rows * case["vocab"]}
    row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * WIDTH[case["cache"]]
    if case["op"] == "compact":
        kept = case["batch"] * (1 + case["kept"] * (case["drafts"] - 1))
        # (the first stays where it is)
        return {"bytes": 2 * row * (kept - case["batch"]) + 4 * case["batch"] * case["drafts"],
                "flops": 0}
    return {"bytes": 2 * row * case["page"] * case["count"] + 8 * case["count"], "flops": 0}
