"""The host side of generation over a paged cache (page pool, room for tokens,
rows that have ended): CPU tests; the model's layers are stood in for."""
import random

import pytest
import torch


def named(pool, seq):
    """The pages that a sequence's row of the table names."""
    return [p for p in pool.table[seq].tolist() if p >= 0]


def test_table_names_only_owned_pages():
    """Whatever is reserved and released, a row names the pages its sequence owns, in
    order, and no others: an entry that names another's page lets a sequence
    write over that one's keys."""
    from cuda_transformer_b200.generate_case import PagePool

    pool = PagePool(6, 4, 2, 4, "cpu")
    assert named(pool, 0) == named(pool, 1) == []
    for seq, tokens in ((0, 16), (1, 4), (0, None), (1, 12), (0, 4)):
        pool.release(seq) if tokens is None else pool.reserve(seq, tokens)
    assert named(pool, 0) == pool.owned[0] and named(pool, 1) == pool.owned[1]

    rng = random.Random(1)
    pool = PagePool(40, 3, 5, 12, "cpu")
    for _ in range(300):
        seq = rng.randrange(5)
        if rng.random() < 0.3:
            pool.release(seq)
        else:
            try:
                pool.reserve(seq, rng.randrange(1, 37))
            except RuntimeError:
                pass
        for b in range(5):
            row = pool.table[b].tolist()
            assert row == pool.owned[b] + [-1] * (12 - len(pool.owned[b]))
        held = sum(pool.owned, [])
        assert len(set(held)) == len(held) and len(held) + len(pool.free) == 40


def generator(batch=2, max_len=8, page=3):
    """A Generator whose layers do nothing: what is left is its book-keeping."""
    from cuda_transformer_b200.generate_case import Generator
    from cuda_transformer_b200.gpt_case import GPT

    gen = Generator(GPT(1, 64, 2, max_len, 10), batch, max_len, page)
    gen._blocks = lambda x, attend: x
    gen._logits = lambda x: x[0, :, :10]
    return gen


def test_prompts_beyond_the_buffers_are_refused():
    """Pages hold up to 9 tokens here, the history and the position table 8."""
    gen = generator()
    for tokens, room in ((9, 0), (2, 9), (0, 0)):
        with pytest.raises(ValueError):
            gen.prompt(0, torch.zeros(tokens, dtype=torch.int64), room)
    gen.prompt(0, torch.zeros(2, dtype=torch.int64), 8)
    with pytest.raises(ValueError):
        gen.generate([torch.zeros(5, dtype=torch.int64)] * 2, 4)
    with pytest.raises(ValueError):
        gen.generate([torch.zeros(5, dtype=torch.int64)], 2)


def test_steps_stay_within_the_reservation():
    """A step that a sequence has no room for is refused before anything changes; one
    without tokens takes no part in steps."""
    gen = generator()
    gen.prompt(0, torch.arange(2), 8)      # three pages, 8 tokens at most
    gen.prompt(1, torch.arange(4))         # two pages, 6 tokens
    for t in range(2):
        gen.step(torch.tensor([7, 5]))
    before = gen.lens.clone(), gen.history.clone()
    with pytest.raises(ValueError):
        gen.step(torch.tensor([7, 5]))
    assert torch.equal(gen.lens, before[0]) and torch.equal(gen.history, before[1])
    assert gen.history[1].tolist() == [0, 1, 2, 3, 5, 5, 0, 0]
    gen.release(1)
    assert named(gen.pool, 1) == []
    for t in range(4):
        gen.step(torch.tensor([6, 9]))
    assert gen.lens.tolist() == [8, 0]
    assert gen.history[0].tolist() == [0, 1, 7, 7, 6, 6, 6, 6] and 9 not in gen.history[1]
    with pytest.raises(ValueError):
        gen.step(torch.tensor([6, 9]))


def test_replayed_steps_stay_within_the_buffers():
    """The device's part of a step, which a graph can repeat without the host: past the
    last place nothing is written and the length stays."""
    gen = generator()
    gen.prompt(0, torch.arange(7), 8)
    for t in range(4):
        gen._step(torch.tensor([3, 4]))
    assert gen.lens.tolist() == [8, 0] and gen.history[0].tolist() == [0, 1, 2, 3, 4, 5, 6, 3]


def test_what_a_step_passes_to_the_operators(monkeypatch):
    """Sequences that take no part append at position -1 (padding) and attend over none."""
    from cuda_transformer import ops

    gen, seen = generator(), []
    monkeypatch.setattr(ops, "kv_append_", lambda *a, **kw: (seen.append(a[5].tolist()), None))
    monkeypatch.setattr(ops, "paged_attention",
                        lambda q, k, v, table, lens, **kw: (seen.append(lens.tolist()), None))
    gen._blocks = lambda x, attend: (attend(0, x[0], x[0], x[0]), x)[1]
    gen.lens[0] = 3
    gen.live[0] = True
    gen.step(torch.tensor([3, 4]))
    assert seen == [[3, -1], [4, 0]]


def test_a_negative_token_ends_its_sequence():
    gen = generator()
    for seq in range(2):
        gen.prompt(seq, torch.arange(2), 8)
    for idx in ([5, -1], [6, 7], [4, 4]):
        gen.step(torch.tensor(idx))
    assert gen.lens.tolist() == [5, 2] and gen.history[1].tolist() == [0, 1] + [0] * 6
    gen.prompt(1, torch.arange(3), 8)
    gen.step(torch.tensor([1, 2]))
    assert gen.lens.tolist() == [6, 4] and gen.history[1, :4].tolist() == [0, 1, 2, 2]
