"""Measured cases of the token-generation operators.

Three operators of one decoding step: ``kv_append_`` (new keys and values into
a paged cache, with the rotary position embedding on the way),
``paged_attention`` (one new query token per sequence against that cache) and
``logits_process`` (repetition, frequency and presence penalties, token biases
and a grammar's bit mask on the logits).

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
def attention(name, batch, q_heads, kv_heads, dim, low, high, page, act, cache, layout):
    """`low`..`high`: range of the cached lengths, spread over its logarithm."""
    return {"name": name, "op": "attention", "batch": batch, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "low": low, "high": high, "page": page,
            "act": act, "cache": cache, "layout": layout}


def append(name, batch, low, high, step, q_heads, kv_heads, dim, rot, interleaved, page, act,
           cache, layout):
    """`step`: one new token a sequence, at positions low..high; else whole
    prompts of low..high tokens."""
    return {"name": name, "op": "append", "batch": batch, "low": low, "high": high, "step": step,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "interleaved": interleaved, "page": page, "act": act, "cache": cache,
            "layout": layout}


def logits(name, rows, vocab, low, high, bias, mask, act):
    """`low`..`high`: range of the history lengths; `bias`: token biases a row."""
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "low": low, "high": high,
            "bias": bias, "mask": mask, "act": act}


def listed():
    return [
        # the character GPT (6 heads of 64, context 256) answering a few prompts: latency
        attention("attn_char_gpt", 8, 6, 6, 64, 1, 256, 16, "f32", "f32", "head"),
        # a busy server: many conversations of very different lengths, grouped heads
        attention("attn_serve_bf16", 64, 32, 8, 128, 16, 4096, 16, "bf16", "bf16", "token"),
        # one long document: few rows, so the cache's length has to be split
        attention("attn_long_bf16", 1, 32, 8, 128, 131072, 131072, 64, "bf16", "bf16", "token"),
        # the FP32 model's heads (32 of 64) over a half-width cache, full batch
        attention("attn_f32_bf16cache", 16, 32, 32, 64, 3500, 4096, 32, "f32", "bf16", "head"),
        # FP32 throughout, pages of an odd size
        attention("attn_f32_odd", 5, 8, 8, 128, 777, 4097, 13, "f32", "f32", "head"),
        # all query heads on one key/value head, f16
        attention("attn_mqa_f16", 128, 16, 1, 64, 1, 16384, 128, "f16", "f16", "token"),
        # a decoding step's new tokens: latency
        append("append_step", 64, 1, 512, True, 32, 8, 128, 128, False, 16, "bf16", "bf16",
               "token"),
        # prompts of a batch, FP32 model into a half-width cache
        append("append_prompts", 12, 300, 4096, False, 32, 32, 64, 64, False, 32, "f32", "bf16",
               "head"),
        # FP32 cache, interleaved pairs, half of the head rotated, pages of an odd size
        append("append_partial_f32", 7, 100, 2000, False, 8, 8, 128, 64, True, 13, "f32", "f32",
               "head"),
        # one answer of the 100256-token GPT: latency
        logits("logits_one", 1, 100256, 256, 256, 16, False, "f32"),
        # a server's step: long histories, biases and a grammar mask
        logits("logits_serve", 256, 100256, 64, 8192, 64, True, "f32"),
        # half-width logits of an odd vocabulary
        logits("logits_odd_bf16", 33, 50257, 1, 2048, 0, True, "bf16"),
    ]


def spread(rng, low, high):
    """A whole number of low..high, uniform over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "logits"])
    act, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                             ("f16", "f16")])
    layout, page = rng.choice(["head", "token"]), rng.choice([1, 8, 13, 16, 24, 32, 64, 128, 256])
    dim = rng.choice([32, 64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 16, 32])
    q_heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 5, 8, 16) if g * kv_heads <= 64])
    if op == "attention":
        # at most 2**28 bytes in each of K and V, as the largest listed cases
        tokens = 2 ** 28 // (kv_heads * dim * WIDTH[cache])
        high = spread(rng, 1, min(131072, tokens))
        batch = spread(rng, 1, max(1, min(512, tokens // high)))
        c = attention("", batch, q_heads, kv_heads, dim, spread(rng, 1, high), high, page, act,
                      cache, layout)
    elif op == "append":
        rot = rng.choice([0, dim // 4, dim // 2, dim, dim])
        step = rng.random() < 0.5
        tokens = 2 ** 24 // (q_heads * dim)
        high = spread(rng, 1, 512 if step else min(8192, tokens))
        batch = spread(rng, 1, 512 if step else max(1, min(64, tokens // high)))
        c = append("", batch, spread(rng, 1, high), high, step, q_heads, kv_heads, dim, rot,
                   rng.random() < 0.3, page, act, cache, layout)
    else:
        vocab = spread(rng, 65, 200000)
        rows = spread(rng, 1, min(256, 25000000 // vocab))
        high = spread(rng, 1, 8192)
        c = logits("", rows, vocab, spread(rng, 1, high), high, rng.choice([0, 0, 1, 16, 64, 300]),
                   rng.random() < 0.5, rng.choice(["f32", "f32", "bf16", "f16"]))
    c.pop("name")
    return c


def lengths(case, count):
    """The case's lengths, the same for every seed: low..high, evenly over the logarithm."""
    low, high = case["low"], case["high"]
    if count == 1:
        return [high]
    return [min(high, max(low, round(low * (high / low) ** (i / (count - 1)))))
            for i in range(count)]


# ------------------------------------------------------------------ inputs
def rotation(positions, rot, device):
    """cos and sin of position * 10000^(-2i/rot), formed in 64 bits, kept in 32."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


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


def cache_pair(case, pool, gen, device):
    """Key and value caches, indexed [page, head, slot, dim]; "token" keeps the
    heads of one token together in memory, "head" the slots of one head."""
    h, s, d, kind = case["kv_heads"], case["page"], case["dim"], DTYPES[case["cache"]]
    shape = (pool, s, h, d) if case["layout"] == "token" else (pool, h, s, d)
    pair = [torch.randn(shape, generator=gen, device=device, dtype=kind) for _ in range(2)]
    return [t.transpose(1, 2) if case["layout"] == "token" else t for t in pair]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    order = random.Random(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)

    state = {"case": case}
    if case["op"] == "attention":
        lens = lengths(case, case["batch"])
        order.shuffle(lens)
        table, pool = page_table(lens, case["page"], gen, device)
        state["k_cache"], state["v_cache"] = cache_pair(case, pool, gen, device)
        state["table"] = table
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
        state["q"] = normal(case["batch"], case["q_heads"], case["dim"]).to(DTYPES[case["act"]])
        # a server keeps one workspace for all its steps (cleared once)
        state["workspace"] = torch.zeros(1 << 23, dtype=torch.uint8, device=device)
    elif case["op"] == "append":
        lens = lengths(case, case["batch"])
        order.shuffle(lens)
        table, pool = page_table(lens, case["page"], gen, device)
        state["k_cache"], state["v_cache"] = cache_pair(case, pool, gen, device)
        state["table"] = table
        if case["step"]:
            state["seq_ids"] = torch.arange(len(lens), dtype=torch.int32, device=device)
            state["positions"] = torch.tensor([n - 1 for n in lens], dtype=torch.int32,
                                              device=device)
        else:
            state["seq_ids"] = torch.cat([torch.full((n,), b, dtype=torch.int32)
                                          for b, n in enumerate(lens)]).to(device)
            state["positions"] = torch.cat([torch.arange(n, dtype=torch.int32)
                                            for n in lens]).to(device)
        # q, k and v are views of one fused projection, as the GPT's blocks make them
        tokens, kind = state["positions"].numel(), DTYPES[case["act"]]
        h = case["q_heads"] + 2 * case["kv_heads"]
        qkv = normal(tokens, h, case["dim"]).to(kind)
        state["q"], state["k"], state["v"] = qkv.split(
            [case["q_heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        state["cos"], state["sin"] = (rotation(case["high"], case["rot"], device) if case["rot"]
                                      else (None, None))
    else:
        rows, vocab = case["rows"], case["vocab"]
        lens = lengths(case, rows)
        order.shuffle(lens)
        # logits of a trained model are a few units wide; ids repeat as words do
        state["logits"] = (3.0 * normal(rows, vocab)).to(DTYPES[case["act"]])
        width = max(lens)
        u = torch.rand(rows, width, generator=gen, device=device, dtype=torch.float64)
        state["tokens"] = (vocab ** u - 1).long().clamp_(0, vocab - 1)
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
        state["prompt_lens"] = (state["lens"].float() *
                                torch.rand(rows, generator=gen, device=device)).int()
        pick = torch.rand(3, rows, generator=gen, device=device)
        state["repetition"] = 1.0 + 0.5 * pick[0]
        state["frequency"], state["presence"] = 0.6 * pick[1], 0.8 * pick[2] - 0.2
        state["bias_ids"] = state["bias_values"] = state["mask"] = None
        if case["bias"]:
            state["bias_ids"] = torch.randint(0, vocab, (rows, case["bias"]), generator=gen,
                                              device=device)
            state["bias_values"] = 4.0 * normal(rows, case["bias"])
        if case["mask"]:
            # runs of allowed and forbidden ids: most words are all or nothing
            words = -(-vocab // 32)
            mixed = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=gen, device=device)
            kind = torch.randint(0, 4, (rows, words), generator=gen, device=device)
            state["mask"] = torch.where(kind == 0, mixed, torch.where(kind == 1, 0, -1)).int()
    return state


# -------------------------------------------------------------------- runs
def run(state):
    return (run_own if own else run_plain)[state["case"]["op"]](state)


def own_attention(s):
    from cuda_transformer import ops

    return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                               workspace=s["workspace"])


def own_append(s):
    from cuda_transformer import ops

    q, _ = ops.kv_append_(s["k_cache"], s["v_cache"], s["k"], s["v"], s["table"], s["positions"],
                          seq_ids=s["seq_ids"], q=s["q"], cos=s["cos"], sin=s["sin"],
                          interleaved=s["case"]["interleaved"])
    return q, s["k_cache"], s["v_cache"]


def own_logits(s):
    from cuda_transformer import ops

    return ops.logits_process(s["logits"], tokens=s["tokens"], lens=s["lens"],
                              prompt_lens=s["prompt_lens"], repetition=s["repetition"],
                              frequency=s["frequency"], presence=s["presence"],
                              bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                              mask=s["mask"])


def plain_attention(s):
    q, table = s["q"].float(), s["table"].long()
    batch, heads, dim = q.shape
    kv = s["k_cache"].shape[1]
    k, v = (c[table].float().transpose(1, 2).reshape(batch, kv, -1, dim)
            for c in (s["k_cache"], s["v_cache"]))
    scores = q.reshape(batch, kv, heads // kv, dim) @ k.transpose(2, 3) * dim ** -0.5
    there = torch.arange(k.shape[2], device=q.device) < s["lens"][:, None]
    scores = torch.where(there[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = top + torch.log(total)
    return out.reshape(batch, heads, dim).to(s["q"].dtype), lse.reshape(batch, heads)


def plain_rotate(x, cos, sin, interleaved):
    x = x.float()
    if cos is None:
        return x
    rot = 2 * cos.shape[1]
    c, n = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def plain_append(s):
    at, page = s["positions"].long(), s["case"]["page"]
    cos, sin = (None, None) if s["cos"] is None else (s["cos"][at], s["sin"][at])
    pages, slots = s["table"][s["seq_ids"].long(), at // page].long(), at % page
    turn = s["case"]["interleaved"]
    q = plain_rotate(s["q"], cos, sin, turn).to(s["q"].dtype)
    s["k_cache"][pages, :, slots] = plain_rotate(s["k"], cos, sin, turn).to(s["k_cache"].dtype)
    s["v_cache"][pages, :, slots] = s["v"].to(s["v_cache"].dtype)
    return q, s["k_cache"], s["v_cache"]


def plain_logits(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    seen = (at < s["lens"][:, None]).float()
    made = seen * (at >= s["prompt_lens"][:, None])
    seen, made = (torch.zeros_like(x).scatter_add_(1, s["tokens"], w) for w in (seen, made))
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * made - s["presence"][:, None] * (made > 0)
    if s["bias_ids"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"], s["bias_values"])
    if s["mask"] is not None:
        ids = torch.arange(vocab, device=x.device)
        x = torch.where((s["mask"][:, ids // 32] >> (ids % 32)) & 1 != 0, x, -math.inf)
    return x


run_own = {"attention": own_attention, "append": own_append, "logits": own_logits}
run_plain = {"attention": plain_attention, "append": plain_append, "logits": plain_logits}


# ------------------------------------------------------------------- exact
def exact_attention(s):
    outs, lses = [], []
    group = s["q"].shape[1] // s["k_cache"].shape[1]
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // s["case"]["page"])].long()
        k, v = (c[pages].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
                for c in (s["k_cache"], s["v_cache"]))
        q = s["q"][b].double().unflatten(0, (-1, group))
        z = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(q.shape[-1])
        outs.append(torch.einsum("hgn,hnd->hgd", z.softmax(-1), v).flatten(0, 1))
        lses.append(z.logsumexp(-1).flatten())
    return torch.stack(outs), torch.stack(lses)


def exact_append(s):
    case = s["case"]
    at = s["positions"].long()

    def turned(x):
        x = x.double()
        if not case["rot"]:
            return x
        half = case["rot"] // 2
        # the pair (a, b) as a + ib, times cos + i sin (the table is an input)
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]
        x = x.clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    pages = s["table"][s["seq_ids"].long(), (at // case["page"])].long()
    k_cache[pages, :, at % case["page"]] = turned(s["k"])
    v_cache[pages, :, at % case["page"]] = s["v"].double()
    return turned(s["q"]), k_cache, v_cache


def exact_logits(s):
    x = s["logits"].double()
    vocab = x.shape[1]
    for i in range(x.shape[0]):
        n, m = int(s["lens"][i]), int(s["prompt_lens"][i])
        there = s["tokens"][i, :n].bincount(minlength=vocab) > 0
        counts = s["tokens"][i, m:n].bincount(minlength=vocab).double()
        r = s["repetition"][i].double()
        x[i] = torch.where(there, torch.maximum(x[i], 0 * x[i]) / r + torch.minimum(x[i], 0 * x[i]) * r,
                           x[i])
        x[i] -= s["frequency"][i].double() * counts + s["presence"][i].double() * counts.clamp(max=1)
        if s["bias_ids"] is not None:
            x[i].index_add_(0, s["bias_ids"][i], s["bias_values"][i].double())
        if s["mask"] is not None:
            bits = (s["mask"][i][:, None] >> torch.arange(32, device=x.device)) & 1
            x[i].masked_fill_(bits.flatten()[:vocab] == 0, -math.inf)
    return x


def exact(case, seed):
    calls = {"attention": exact_attention, "append": exact_append, "logits": exact_logits}
    return calls[case["op"]](prepare(case, seed))


# -------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attention":
        total = sum(lengths(case, case["batch"]))
        rows = case["batch"] * case["q_heads"]
        group = case["q_heads"] // case["kv_heads"]
        values = total * case["kv_heads"] * case["dim"]
        pages = sum(-(-n // case["page"]) for n in lengths(case, case["batch"]))
        moved = 2 * values * WIDTH[case["cache"]] + 2 * rows * case["dim"] * WIDTH[case["act"]]
        return {"bytes": moved + 4 * rows + 4 * pages + 4 * case["batch"],
                "flops": 4 * group * values}
    if case["op"] == "append":
        lens = lengths(case, case["batch"])
        tokens = case["batch"] if case["step"] else sum(lens)
        q, kv = case["q_heads"] * case["dim"], case["kv_heads"] * case["dim"]
        angles = 4 * case["rot"] * (tokens if case["step"] else max(lens))
        moved = tokens * ((2 * q + 2 * kv) * WIDTH[case["act"]] + 2 * kv * WIDTH[case["cache"]] + 8)
        turned = tokens * (case["q_heads"] + case["kv_heads"]) * case["rot"]
        return {"bytes": moved + angles, "flops": 3 * turned}
    lens = lengths(case, case["rows"])
    values = case["rows"] * case["vocab"]
    moved = values * (WIDTH[case["act"]] + 4) + 8 * sum(lens) + case["rows"] * 20
    moved += case["rows"] * case["bias"] * 12 + (values // 8 if case["mask"] else 0)
    return {"bytes": moved, "flops": 4 * values}
