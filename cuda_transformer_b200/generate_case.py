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

Prompts that are given several times run once and are forked: kv_copy_pages_
copies the page that is not full, the others are shared.  With --drafts a step
feeds a small tree of tokens instead of one: what followed the last token
where it came up before.  tree_attention looks at all of them, verify_drafts
keeps a path, kv_compact_ moves its keys and values to where the next step
expects them.

  python -m cuda_transformer_b200.generate_case [--batch 8 --new 128 --graph]
      [--cache bf16] [--rotary] [--temperature 0.8 --repetition 1.1] [--check]
      [--samples 4] [--drafts 4 --branches 2]

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
    sequence the pages for `tokens` tokens, `release` takes them back, `fork`
    lets one begin with another's.  A row names the pages that its sequence
    owns and is -1 past them, which the operators take for no place: a token
    too many gives NaN there and does not reach another sequence's pages."""

    def __init__(self, pages: int, page_size: int, batch: int, max_pages: int, device):
        self.page_size, self.max_pages = page_size, max_pages
        self.free = list(range(pages - 1, -1, -1))
        self.owned: list[list[int]] = [[] for _ in range(batch)]
        self.users = [0] * pages  # sequences that have a page
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
            for page in new:
                self.users[page] += 1
            self.table[seq, at:need] = torch.tensor(new, dtype=torch.int32)

    def release(self, seq: int) -> None:
        for page in reversed(self.owned[seq]):
            self.users[page] -= 1
            if self.users[page] == 0:
                self.free.append(page)
        self.owned[seq] = []
        self.table[seq] = -1

    def fork(self, src: int, dst: int, tokens: int) -> list[tuple[int, int]]:
        """Sequence dst, which has no pages, begins with the first `tokens`
        tokens of src: it shares the pages that those fill and gets one of its
        own for the rest.  Returns the (from, to) pages to copy: that one."""
        if self.owned[dst]:
            raise ValueError(f"sequence {dst} has pages")
        full, need = tokens // self.page_size, -(-tokens // self.page_size)
        if need > len(self.owned[src]):
            raise ValueError(f"sequence {src} has no {tokens} tokens")
        if need > full and not self.free:
            raise RuntimeError("out of pages: 1 needed, 0 free")
        shared = self.owned[src][:full]
        for page in shared:
            self.users[page] += 1
        self.owned[dst] = list(shared)
        if full:
            self.table[dst, :full] = self.table[src, :full]
        self.reserve(dst, tokens)
        return [(self.owned[src][full], self.owned[dst][full])] if need > full else []


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
        # The host's counts of the tokens (0: none begun).  keep_path adds up to _ahead
        # tokens that they lack; a graph that holds one does so unseen.
        self.counts, self._ahead, self._captured = [0] * batch, 0, False

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

    def fork(self, src: int, dst: int, room: int = 0) -> None:
        """Sequence dst begins as src is now (its tokens and their cached keys
        and values); `room`: tokens to reserve pages for."""
        self._count()
        n = self.counts[src]
        if n == 0 or src == dst:
            raise ValueError(f"sequence {src} cannot be forked into {dst}")
        if max(n, room) > self.max_len:
            raise ValueError(f"{max(n, room)} tokens are more than max_len, {self.max_len}")
        self.release(dst)
        pairs = self.pool.fork(src, dst, n)
        try:
            self.pool.reserve(dst, max(n, room))
        except (RuntimeError, ValueError):
            self.release(dst)
            raise
        if pairs:
            pages = torch.tensor(pairs, dtype=torch.int32, device=self.history.device)
            ops.kv_copy_pages_([c for pair in self.caches for c in pair], pages[:, 0], pages[:, 1])
        for t in (self.history, self.lens, self.prompt_lens, self.live):
            t[dst] = t[src]
        self.counts[dst] = n

    def step(self, idx: torch.Tensor) -> torch.Tensor:
        """Feeds one token a sequence (int64 [batch]; their places are the
        current lengths) and returns the logits after them [batch, vocab]
        (those of sequences that take no part mean nothing).  A negative token
        ends its sequence; its pages stay until `release`.  No host
        synchronisation, unless room is short after `keep_path`: then the
        lengths are read back.  A sequence without room for it is a ValueError."""
        self._take_room()
        return self._step(idx)

    def _count(self) -> None:
        """Brings the host's counts up to the device's."""
        if self._ahead or self._captured:
            self.counts = [have if n else 0 for n, have in zip(self.counts, self.lens.tolist())]
            self._ahead = 0

    def _need_room(self, more: int) -> None:
        if self._captured:
            self._count()
        while True:
            full = [seq for seq, n in enumerate(self.counts) if n and n + self._ahead + more > min(
                self.max_len, len(self.pool.owned[seq]) * self.pool.page_size)]
            if full and not self._ahead:
                raise ValueError(f"sequence {full[0]} has no room for {more} more tokens after its "
                                 f"{self.counts[full[0]]}")
            if not full:
                return
            self._count()

    def _take_room(self) -> None:
        self._need_room(1)
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

    def _probabilities(self, logits: torch.Tensor, temperature: float) -> torch.Tensor:
        # (bounded: +inf, as a bias can make it, takes all of the softmax)
        top = torch.finfo(torch.float32).max
        return ops.cuda_softmax((logits / temperature).clamp_(max=top))

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
            probs = self._probabilities(logits.unsqueeze(0), temperature)[0]
            # the first token whose running sum passes the number; a scan's sums can
            # step up by a rounding at a token of probability 0, which has no say
            upto = torch.where(probs > 0, probs.cumsum(-1), 0.0)
            total = upto.amax(-1)
            idx = (upto > (uniform * total)[:, None]).int().argmax(-1)
            there = total > 0
        return torch.where(there & self.live, idx, -1)

    def _prompts(self, prompts, room: int) -> torch.Tensor:
        """Begins all sequences, with pages for `room` tokens after their
        prompts; the logits after them [batch, vocab]."""
        logits: list[torch.Tensor] = []
        for b, t in enumerate(prompts):
            same = next((i for i in range(b) if prompts[i] is t), None)
            if same is None:
                logits.append(self.prompt(b, t, t.numel() + room))
            else:
                self.fork(same, b, t.numel() + room)
                logits.append(logits[same])
        return torch.stack(logits)

    def look_up_drafts(self, root: torch.Tensor, depth: int, branches: int) -> torch.Tensor:
        """Drafts for the tokens after `root` (int64 [batch], which the history
        does not hold yet): `depth` tokens of what followed it at the last
        `branches` places where it came up before, those first where the token
        before it is the same too.  int64 [batch, 1 + branches * depth]: root,
        then the branches; -1: no token."""
        at = torch.arange(self.max_len, device=root.device)
        lens = self.lens[:, None].long()
        known = at < lens
        there = known & (self.history == root[:, None])
        last = self.history.gather(1, (lens - 1).clamp(min=0))
        alike = torch.zeros_like(there)
        alike[:, 1:] = there[:, 1:] & (self.history[:, :-1] == last)
        rank = torch.where(alike, at + self.max_len, torch.where(there, at, -1))
        best = rank.topk(min(branches, self.max_len), dim=1).values
        places = best.remainder(self.max_len)[:, :, None] + torch.arange(1, depth + 1, device=root.device)
        tokens = self.history.gather(1, places.flatten(1).clamp(max=self.max_len - 1))
        fine = (best >= 0)[:, :, None] & (places < lens[:, :, None])
        return torch.cat([root[:, None], torch.where(fine.flatten(1), tokens, -1)], 1)

    def step_drafts(self, tokens: torch.Tensor, parents: torch.Tensor, mask: torch.Tensor,
                    depths: torch.Tensor) -> torch.Tensor:
        """Feeds every sequence the nodes of a tree (tokens int64 [batch, n],
        node 0 its next token; the tree as verify_drafts and tree_attention
        take it, depths int32 [n] its nodes' distances from node 0) and returns
        the logits after each [batch, n, vocab].  The nodes' keys and values
        are in the cache behind the sequence, in their order; `keep_path` says
        which of them stay.  A sequence without room for n tokens is a
        ValueError (in a graph, whose replays the host does not see: NaN).  A
        negative node 0 ends its sequence, as in `step`."""
        if not (tokens.is_cuda and torch.cuda.is_current_stream_capturing()):
            self._need_room(tokens.shape[1])
        return self._step_drafts(tokens, parents, mask, depths)

    @torch.no_grad()
    def _step_drafts(self, tokens, parents, mask, depths):
        """The device's part of a drafted step."""
        batch, n = tokens.shape
        self.live &= tokens[:, 0] >= 0
        at = torch.arange(n, dtype=torch.int32, device=tokens.device)
        context = torch.where(self.live, self.lens, -1)
        slots = torch.where(self.live[:, None], self.lens[:, None] + at, -1).flatten()
        places = (self.lens[:, None] + depths).clamp(max=self.max_len - 1).flatten()
        ids = torch.arange(batch, dtype=torch.int32, device=tokens.device).repeat_interleave(n)

        def attend(layer, q, k, v):
            q2, _ = ops.kv_append_(*self.caches[layer], k, v, self.pool.table, slots, seq_ids=ids,
                                   q=q if self.rotary else None, cos=self.cos, sin=self.sin,
                                   rotary_positions=places if self.rotary else None)
            q = (q2 if self.rotary else q).unflatten(0, (batch, n))
            o, _ = ops.tree_attention(q, *self.caches[layer], self.pool.table, context, mask=mask)
            return o.flatten(0, 1)

        x = self._embed(tokens.flatten().clamp(min=0), places).unsqueeze(0)
        return self._logits(self._blocks(x, attend)).unflatten(0, (batch, n))

    @torch.no_grad()
    def keep_path(self, tokens: torch.Tensor, path: torch.Tensor, counts: torch.Tensor) -> None:
        """The nodes of `path` (verify_drafts') join their sequences, in the
        cache and in the history.  How many, the host learns when it has to
        know (`fork`)."""
        self._ahead += path.shape[1]
        if path.is_cuda and torch.cuda.is_current_stream_capturing():
            self._captured = True
        counts = torch.where(self.live, counts, 0)
        counts = torch.minimum(counts, self.max_len - self.lens)  # (what has no column)
        ops.kv_compact_([c for pair in self.caches for c in pair], self.pool.table, self.lens, path,
                        counts)
        at = torch.arange(path.shape[1], device=path.device)
        kept = at < counts[:, None]
        column = torch.where(kept, self.lens[:, None] + at, self.max_len)
        self._columns.scatter_(1, column.long(), tokens.gather(1, path.clamp(min=0).long()))
        self.lens += counts

    def generate_drafted(self, prompts, new: int, depth: int = 4, branches: int = 1,
                         temperature: float = 0.0, seed: int = 0):
        """`new` tokens after each prompt [batch, new], as generate gives them
        without processing (with a temperature: distributed alike), and the
        number of steps that it took.  Each step feeds a tree of looked-up
        tokens; max_len has to hold branches * depth tokens more than the
        prompts and the new ones.  A sequence that has no next token ends: -1.
        The others go on from there: they hold all of their tokens but the
        last, which the next `step` feeds."""
        if len(prompts) != self.batch:
            raise ValueError(f"{len(prompts)} prompts for {self.batch} sequences")
        if depth < 0 or branches < 0:
            raise ValueError(f"drafts of {branches} branches of {depth} tokens")
        device = self.history.device
        n = 1 + branches * depth
        span = max(depth, 1)  # (a tree may be its root alone)
        node = torch.arange(n, dtype=torch.int32, device=device)
        first = (node - 1) % span == 0
        parents = torch.where(node == 0, -1, torch.where(first, 0, node - 1))
        depths = torch.where(node == 0, 0, (node - 1) % span + 1).int()
        # a node sees the root and its branch up to itself
        alike = (node[:, None] - 1) // span == (node - 1) // span
        sees = (node == 0) | (alike & (node <= node[:, None]) & (node[:, None] > 0))
        words = torch.nn.functional.pad(sees, (0, -n % 32)).unflatten(1, (-1, 32)).long()
        words = (words << torch.arange(32, device=device)).sum(-1)
        mask = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
        mask = mask.expand(self.batch, n, mask.shape[1])
        parents = parents.int().expand(self.batch, n)
        g = torch.Generator(device=device).manual_seed(seed)

        def uniform():
            return torch.rand(self.batch, n, generator=g, device=device) if temperature else None

        def scores(logits):  # what verify_drafts takes: scores, or probabilities
            return logits if temperature == 0.0 else self._probabilities(logits, temperature)

        logits = self._prompts(prompts, new + n)
        begun = list(self.counts)
        # the first token: a tree of its root alone
        u = uniform()
        root = ops.verify_drafts(scores(logits[:, None]), torch.zeros_like(self.lens)[:, None].long(),
                                 uniform=None if u is None else u[:, :1])[0][:, 0]
        made = [[] for _ in prompts]
        steps, roots = 0, root.tolist()
        for seq, token in enumerate(roots):
            made[seq].append(token)
        while True:
            ended = [len(m) >= new or m[-1] < 0 for m in made]
            if all(ended):
                break
            self.live &= ~torch.tensor(ended, device=device)
            tokens = self.look_up_drafts(root, depth, branches)
            logits = self._step_drafts(tokens, parents, mask, depths)
            found, path, counts = ops.verify_drafts(scores(logits), tokens, parents,
                                                    uniform=uniform())
            self.keep_path(tokens, path, counts)
            root = found.gather(1, (counts - 1).clamp(min=0).long()[:, None])[:, 0]
            steps += 1
            for seq, (row, count) in enumerate(zip(found.tolist(), counts.tolist())):
                if not ended[seq]:
                    made[seq].extend(row[:count])
        # what came after the last token goes out again (no row reads it)
        there = [(m + [-1]).index(-1) for m in made]
        fed = [n + min(t, max(new - 1, 0)) for n, t in zip(begun, there)]
        self.lens.copy_(torch.tensor(fed, dtype=torch.int32))
        self.live.copy_(torch.tensor([t >= new for t in there]))
        self.counts, self._ahead = fed, 0
        filled = [(m + [-1] * new)[:new] for m in made]
        return torch.tensor(filled, device=device), steps

    def generate(self, prompts, new: int, temperature: float = 0.0, seed: int = 0,
                 graph: bool = False, **processing):
        """`new` tokens after each prompt; returns them [batch, new] and the
        unprocessed logits that each was chosen from [new, batch, vocab].  A
        sequence that has no next token ends: -1 from there on.  A prompt that
        is in the list several times (one tensor) runs once and is forked."""
        if len(prompts) != self.batch:
            raise ValueError(f"{len(prompts)} prompts for {self.batch} sequences")
        g = torch.Generator(device=self.history.device).manual_seed(seed)
        uniform = torch.rand(new, self.batch, generator=g, device=self.history.device)
        logits = self._prompts(prompts, new)
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
    ap.add_argument("--samples", type=int, default=1, help="answers to each prompt (forked)")
    ap.add_argument("--drafts", type=int, default=0, help="looked-up tokens a branch and step")
    ap.add_argument("--branches", type=int, default=1)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    torch.cuda.set_device(dev)
    torch.manual_seed(1234)
    model = GPT(a.layers, a.d, a.heads, a.ctx, a.vocab).to(dev)
    g = torch.Generator().manual_seed(7)
    nodes = 1 + a.drafts * a.branches if a.drafts else 0
    most = a.ctx - a.new - nodes
    if a.drafts and (a.graph or a.repetition != 1.0 or a.frequency or a.presence):
        ap.error("--drafts goes without --graph and without penalties")
    if most < 1 or a.batch % a.samples:
        ap.error("--ctx must hold a prompt and the new tokens, --batch whole groups of --samples")
    prompts = [torch.randint(0, a.vocab, (int(n),), generator=g).to(dev)
               for n in torch.randint(1, most + 1, (a.batch // a.samples,), generator=g)]
    prompts = [p for p in prompts for _ in range(a.samples)]
    gen = Generator(model, a.batch, a.ctx, a.page, CACHE_TYPES[a.cache], a.rotary)
    full = lambda x: torch.full((a.batch,), x, device=dev)  # noqa: E731
    args = dict(temperature=a.temperature, graph=a.graph, repetition=full(a.repetition),
                frequency=full(a.frequency), presence=full(a.presence))

    def run(new):
        if a.drafts:
            return gen.generate_drafted(prompts, new, a.drafts, a.branches, a.temperature)
        return gen.generate(prompts, new, **args)

    run(min(a.new, 4))  # warm-up
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    tokens, logits = run(a.new)
    torch.cuda.synchronize()
    took = time.perf_counter() - t0
    line = {"metric": "GPT generation tokens/s", "value": a.batch * a.new / took,
            "unit": "tokens/s", "ms_per_token": took / a.new * 1e3, "batch": a.batch,
            "new_tokens": a.new, "prompt_lens": [t.numel() for t in prompts],
            "config": {"layers": a.layers, "d_model": a.d, "heads": a.heads, "vocab": a.vocab,
                       "page": a.page, "cache": a.cache, "rotary": a.rotary, "graph": a.graph},
            "data": "random prompts and weights; prompts included in the time"}
    if a.drafts:
        steps, logits = logits, None
        line["steps"] = steps
        line["config"] |= {"drafts": a.drafts, "branches": a.branches}
    if a.check and a.drafts:  # how far below the best one a chosen token's logit is
        worst = 0.0
        for b, p in enumerate(prompts):
            seq = torch.cat([p, tokens[b]])
            for t in range(a.new):
                ref = whole_sequence_logits(model, seq[:p.numel() + t], a.rotary)
                worst = max(worst, (ref.max() - ref[tokens[b, t]]).item())
        line["below_best_logit"] = worst
    elif a.check:
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
