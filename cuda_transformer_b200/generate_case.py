"""Token generation with the GPT of gpt_case over a paged key/value cache.

Prompts run through the model's FlashAttention-2 forward, and kv_append_ puts
their keys and values into the cache; after that every step feeds one token a
sequence: kv_append_ writes its keys and values, paged_attention attends over
the cache, logits_process applies the repetition, frequency and presence
penalties, biases and grammar mask, and the next token is the best one or is
drawn from the softmax (the reference's GPT.generate draws from the softmax of
the last logits, gpt/gpt.py:184, and keeps no cache).  Sequences have lengths
of their own.  With --rotary the learned position table gives way to rotary
embeddings.  The steps can run from a CUDA graph: nothing in a step depends on
a value that the host would have to read.

  python -m cuda_transformer_b200.generate_case [--batch 8 --new 128 --graph]
      [--cache bf16] [--rotary] [--temperature 0.8 --repetition 1.1] [--check]

--check generates the same tokens again by running every whole sequence through
the model at each step, and compares the logits.  Prints one JSON line.
"""
from __future__ import annotations

import argparse
import json
import time

import torch

from cuda_transformer import ops

from .gpt_case import GPT, CudaFlashAttention, CudaLinearLayer, CudaMLP

CACHE_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


class PagePool:
    """Which pages of a cache belong to which sequence (host side).  table is
    the int32 [batch, max_pages] that the operators read; `reserve` gives a
    sequence the pages for `tokens` tokens, `release` takes them back.  A row
    names the pages that its sequence owns and is -1 past them, which the
    operators take for no place: a token too many gives NaN there and does not
    reach another sequence's pages."""

    def __init__(self, pages: int, page_size: int, batch: int, max_pages: int, device):
        self.page_size, self.max_pages = page_size, max_pages
        self.free = list(range(pages - 1, -1, -1))
        self.owned: list[list[int]] = [[] for _ in range(batch)]
        self.table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)

    def reserve(self, seq: int, tokens: int) -> None:
        have, need = self.owned[seq], -(-tokens // self.page_size)
        if need > self.max_pages:
            raise ValueError(f"{tokens} tokens need {need} pages, the table has {self.max_pages}")
        if need - len(have) > len(self.free):
            raise RuntimeError(f"out of pages: {need - len(have)} needed, {len(self.free)} free")
        if need > len(have):
            new = [self.free.pop() for _ in range(need - len(have))]
            at = len(have)
            have.extend(new)
            self.table[seq, at:need] = torch.tensor(new, dtype=torch.int32)

    def release(self, seq: int) -> None:
        self.free.extend(reversed(self.owned[seq]))
        self.owned[seq] = []
        self.table[seq] = -1


class Generator:
    """Generates from a GPT for `batch` sequences of up to `max_len` tokens.
    `prompt` begins a sequence, `release` ends it; in between every `step` feeds
    it a token.  Sequences that have not begun or have ended take no part."""

    def __init__(self, model: GPT, batch: int, max_len: int, page_size: int = 16,
                 cache: torch.dtype = torch.float32, rotary: bool = False):
        self.model, self.batch, self.max_len = model, batch, max_len
        self.rotary = rotary
        device = model.tok.weight.device
        heads, hs = model.blocks[0].attn.heads, model.blocks[0].attn.hs
        if not rotary and max_len > model.pos.weight.shape[0]:
            raise ValueError("max_len is beyond the model's position table")
        max_pages = -(-max_len // page_size)
        self.pool = PagePool(batch * max_pages, page_size, batch, max_pages, device)
        shape = (batch * max_pages, heads, page_size, hs)
        self.caches = [tuple(torch.zeros(shape, dtype=cache, device=device) for _ in range(2))
                       for _ in model.blocks]
        self.workspace = ops.paged_attention_workspace(heads, heads, hs, device)
        self.cos, self.sin = (ops.rotary_tables(max_len, hs, device=device) if rotary
                              else (None, None))
        # one column more than is read: where tokens without a place are written
        self._columns = torch.zeros(batch, max_len + 1, dtype=torch.int64, device=device)
        self.history = self._columns[:, :max_len]
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)  # tokens in the history
        self.prompt_lens = torch.zeros_like(self.lens)
        self.live = torch.zeros(batch, dtype=torch.bool, device=device)  # takes part in steps
        self.counts = [0] * batch  # the host's count of the tokens; 0: none begun

    def _embed(self, idx, positions):
        x = self.model.tok(idx)
        return x if self.rotary else x + self.model.pos(positions)

    def _blocks(self, x, attend):
        """The model's blocks on x [1, tokens, d]; attend(layer, q, k, v) on
        [tokens, heads, hs] views gives [tokens, d]."""
        for layer, blk in enumerate(self.model.blocks):
            qkv = CudaLinearLayer.apply(blk.ln1(x), blk.attn.qkv_weight, blk.attn.qkv_bias)
            q, k, v = qkv[0].view(-1, 3, blk.attn.heads, blk.attn.hs).unbind(1)
            o = attend(layer, q, k, v).reshape(x.shape)
            x = x + CudaLinearLayer.apply(o, blk.attn.out_weight, blk.attn.out_bias)
            m = blk.mlp
            x = x + CudaMLP.apply(blk.ln2(x), m.fc1_weights, m.fc1_bias, m.fc2_weights, m.fc2_bias)
        return x

    def _logits(self, x):
        m = self.model
        w = m.tok.weight.t() if m.tied else m.lm_head_weights
        return CudaLinearLayer.apply(m.ln(x), w, m.lm_head_bias)[0]

    def release(self, seq: int) -> None:
        """Ends a sequence and gives its pages back."""
        self.pool.release(seq)
        self.live[seq] = False
        self.lens[seq] = self.prompt_lens[seq] = 0
        self.counts[seq] = 0

    @torch.no_grad()
    def prompt(self, seq: int, tokens: torch.Tensor, room: int = 0) -> torch.Tensor:
        """Runs a prompt (int64 [n], n > 0) as sequence `seq` and returns the
        logits after it [vocab]; `room`: tokens to reserve pages for."""
        n = tokens.numel()
        if n == 0:
            raise ValueError("a prompt has at least one token")
        if max(n, room) > self.max_len:
            raise ValueError(f"{max(n, room)} tokens are more than max_len, {self.max_len}")
        self.release(seq)
        self.pool.reserve(seq, max(n, room))
        device = self.history.device
        positions = torch.arange(n, dtype=torch.int32, device=device)
        ids = torch.full((n,), seq, dtype=torch.int32, device=device)

        def attend(layer, q, k, v):
            q2, k2 = ops.kv_append_(*self.caches[layer], k, v, self.pool.table, positions,
                                    seq_ids=ids, q=q if self.rotary else None, cos=self.cos,
                                    sin=self.sin, want_k=self.rotary)
            if self.rotary:
                q, k = q2, k2
            o, _ = CudaFlashAttention.apply(*(t.transpose(0, 1).unsqueeze(0) for t in (q, k, v)),
                                            True)
            return o[0].transpose(0, 1)

        x = self._blocks(self._embed(tokens.to(device), positions).unsqueeze(0), attend)
        self.history[seq, :n] = tokens.to(device)
        self.lens[seq] = self.prompt_lens[seq] = self.counts[seq] = n
        self.live[seq] = True
        return self._logits(x[:, -1:])[0]

    def step(self, idx: torch.Tensor) -> torch.Tensor:
        """Feeds one token a sequence (int64 [batch]; their places are the
        current lengths) and returns the logits after them [batch, vocab]
        (those of sequences that take no part mean nothing).  A negative token
        ends its sequence; its pages stay until `release`.  No host
        synchronisation.  A sequence without room for it is a ValueError."""
        self._take_room()
        return self._step(idx)

    def _take_room(self) -> None:
        for seq, n in enumerate(self.counts):
            if n and n >= min(self.max_len, len(self.pool.owned[seq]) * self.pool.page_size):
                raise ValueError(f"sequence {seq} has no room for a token after its {n}")
        self.counts = [n + 1 if n else 0 for n in self.counts]

    @torch.no_grad()
    def _step(self, idx: torch.Tensor) -> torch.Tensor:
        """The device's part of a step."""
        self.live &= idx >= 0
        positions = torch.where(self.live, self.lens, -1)  # -1: padding
        at = self.lens.clamp(max=self.max_len - 1)
        column = positions.remainder(self.max_len + 1).long()
        self._columns.scatter_(1, column[:, None], idx[:, None])
        self.lens += self.live
        self.lens.clamp_(max=self.max_len)
        lens = positions + 1

        def attend(layer, q, k, v):
            q2, _ = ops.kv_append_(*self.caches[layer], k, v, self.pool.table, positions,
                                   q=q if self.rotary else None, cos=self.cos, sin=self.sin)
            o, _ = ops.paged_attention(q2 if self.rotary else q, *self.caches[layer],
                                       self.pool.table, lens, workspace=self.workspace)
            return o

        x = self._embed(idx.clamp(min=0), at).unsqueeze(0)
        return self._logits(self._blocks(x, attend))

    @torch.no_grad()
    def choose(self, logits: torch.Tensor, temperature: float = 0.0, uniform=None,
               **processing) -> torch.Tensor:
        """The next token of each row: the best one, or with a temperature the
        one that `uniform` ([batch] numbers in [0, 1)) draws; -1 for rows without
        one: the mask leaves nothing, the logits are NaN, the sequence takes no
        part.  processing: logits_process's repetition, frequency, presence,
        biases and mask."""
        logits = ops.logits_process(logits, tokens=self.history, lens=self.lens,
                                    prompt_lens=self.prompt_lens, **processing)
        if temperature == 0.0:
            best, idx = logits.max(-1)
            there = best > float("-inf")  # (false for NaN too)
        else:
            # (bounded: +inf, as a bias can make it, takes all of the softmax)
            top = torch.finfo(torch.float32).max
            probs = ops.cuda_softmax((logits / temperature).clamp_(max=top).unsqueeze(0))[0]
            # the first token whose running sum passes the number; a scan's sums can
            # step up by a rounding at a token of probability 0, which has no say
            upto = torch.where(probs > 0, probs.cumsum(-1), 0.0)
            total = upto.amax(-1)
            idx = (upto > (uniform * total)[:, None]).int().argmax(-1)
            there = total > 0
        return torch.where(there & self.live, idx, -1)

    def generate(self, prompts, new: int, temperature: float = 0.0, seed: int = 0,
                 graph: bool = False, **processing):
        """`new` tokens after each prompt; returns them [batch, new] and the
        unprocessed logits that each was chosen from [new, batch, vocab].  A
        sequence that has no next token ends: -1 from there on."""
        if len(prompts) != self.batch:
            raise ValueError(f"{len(prompts)} prompts for {self.batch} sequences")
        g = torch.Generator(device=self.history.device).manual_seed(seed)
        uniform = torch.rand(new, self.batch, generator=g, device=self.history.device)
        logits = torch.stack([self.prompt(b, t, t.numel() + new) for b, t in enumerate(prompts)])
        draw = torch.empty(self.batch, device=uniform.device)
        state = {"logits": logits}

        def advance():
            idx = self.choose(state["logits"], temperature, draw, **processing)
            return idx, self._step(idx)

        replay = None
        if graph:
            # warm up on a side stream (lazy initialisation), then capture; the
            # lengths go back to the prompts' and every step overwrites its slots
            keep, live = self.lens.clone(), self.live.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                draw.fill_(0.5)
                advance()
            torch.cuda.current_stream().wait_stream(side)
            self.lens.copy_(keep)
            self.live.copy_(live)
            replay = torch.cuda.CUDAGraph()
            with torch.cuda.graph(replay):
                held, after = advance()
                state["logits"].copy_(after)
            self.lens.copy_(keep)
        tokens, seen = [], []
        for t in range(new):
            draw.copy_(uniform[t])
            seen.append(state["logits"].clone())
            self._take_room()
            if replay is not None:
                replay.replay()
                tokens.append(held.clone())
            else:
                idx, state["logits"] = advance()
                tokens.append(idx)
        return torch.stack(tokens, 1), torch.stack(seen)


@torch.no_grad()
def whole_sequence_logits(model: GPT, tokens: torch.Tensor, rotary: bool = False) -> torch.Tensor:
    """Logits after the last of `tokens` (int64 [n]) without a cache; rotary
    angles applied with torch."""
    if not rotary:
        return model(tokens[None])[0][0, -1]
    n = tokens.numel()
    cos, sin = ops.rotary_tables(n, model.blocks[0].attn.hs, device=tokens.device)

    def turn(x):  # [n, heads, hs]
        a, b = x.chunk(2, -1)
        c, s = cos[:, None], sin[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    x = model.tok(tokens)[None]
    for blk in model.blocks:
        qkv = CudaLinearLayer.apply(blk.ln1(x), blk.attn.qkv_weight, blk.attn.qkv_bias)
        q, k, v = qkv[0].view(n, 3, blk.attn.heads, blk.attn.hs).unbind(1)
        o, _ = CudaFlashAttention.apply(*(t.transpose(0, 1).unsqueeze(0)
                                          for t in (turn(q), turn(k), v)), True)
        x = x + CudaLinearLayer.apply(o[0].transpose(0, 1).reshape(x.shape), blk.attn.out_weight,
                                      blk.attn.out_bias)
        x = x + blk.mlp(blk.ln2(x))
    w = model.tok.weight.t() if model.tied else model.lm_head_weights
    return CudaLinearLayer.apply(model.ln(x[:, -1:]), w, model.lm_head_bias)[0, 0]


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=6)
    ap.add_argument("--d", type=int, default=384)
    ap.add_argument("--heads", type=int, default=6)
    ap.add_argument("--ctx", type=int, default=256)
    ap.add_argument("--vocab", type=int, default=65)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--new", type=int, default=128, help="tokens to generate after each prompt")
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--cache", default="f32", choices=sorted(CACHE_TYPES))
    ap.add_argument("--rotary", action="store_true")
    ap.add_argument("--graph", action="store_true", help="run the steps from a CUDA graph")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--repetition", type=float, default=1.0)
    ap.add_argument("--frequency", type=float, default=0.0)
    ap.add_argument("--presence", type=float, default=0.0)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    torch.manual_seed(1234)
    model = GPT(a.layers, a.d, a.heads, a.ctx, a.vocab).to(dev)
    g = torch.Generator().manual_seed(7)
    most = a.ctx - a.new
    prompts = [torch.randint(0, a.vocab, (int(n),), generator=g).to(dev)
               for n in torch.randint(1, most + 1, (a.batch,), generator=g)]
    gen = Generator(model, a.batch, a.ctx, a.page, CACHE_TYPES[a.cache], a.rotary)
    full = lambda x: torch.full((a.batch,), x, device=dev)  # noqa: E731
    args = dict(temperature=a.temperature, graph=a.graph, repetition=full(a.repetition),
                frequency=full(a.frequency), presence=full(a.presence))
    gen.generate(prompts, min(a.new, 4), **args)  # warm-up
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens, logits = gen.generate(prompts, a.new, **args)
    torch.cuda.synchronize()
    took = time.perf_counter() - t0
    line = {"metric": "GPT generation tokens/s", "value": a.batch * a.new / took,
            "unit": "tokens/s", "ms_per_token": took / a.new * 1e3, "batch": a.batch,
            "new_tokens": a.new, "prompt_lens": [t.numel() for t in prompts],
            "config": {"layers": a.layers, "d_model": a.d, "heads": a.heads, "vocab": a.vocab,
                       "page": a.page, "cache": a.cache, "rotary": a.rotary, "graph": a.graph},
            "data": "random prompts and weights; prompts included in the time"}
    if a.check:
        worst = 0.0
        for b, p in enumerate(prompts):
            seq = torch.cat([p, tokens[b]])
            for t in range(a.new):
                ref = whole_sequence_logits(model, seq[:p.numel() + t], a.rotary)
                worst = max(worst, (ref - logits[t, b]).abs().max().item())
        line["max_logit_difference"] = worst
    print(json.dumps(line), flush=True)


if __name__ == "__main__":
    main()
