"""What the host knows of a generator's sequences while drafts are kept on the device: CPU
tests (the operators that move what the cache holds are stand-ins)."""
import pytest
import torch


@pytest.fixture
def moved(monkeypatch):
    """Calls of the cache operators, by name."""
    from cuda_transformer_b200 import generate_case

    calls = []
    monkeypatch.setattr(generate_case.ops, "kv_compact_", lambda caches, *a: calls.append(("compact",) + a))
    monkeypatch.setattr(generate_case.ops, "kv_copy_pages_",
                        lambda caches, src, dst: calls.append(("copy", src.tolist(), dst.tolist())))
    return calls


def generator(batch=2, max_len=48, page=4, **kw):
    from cuda_transformer_b200.generate_case import Generator
    from cuda_transformer_b200.gpt_case import GPT

    return Generator(GPT(1, 64, 2, max_len, 10), batch, max_len, page, **kw)


def begin(gen, seq, tokens, room):
    """As `prompt` leaves a sequence."""
    gen.pool.reserve(seq, room)
    gen.history[seq, :tokens] = torch.arange(tokens)
    gen.lens[seq] = gen.prompt_lens[seq] = gen.counts[seq] = tokens
    gen.live[seq] = True


def keep(gen, counts, n=None):
    """keep_path of a chain's first counts[b] nodes."""
    n = n or max(counts)
    at = torch.arange(n, dtype=torch.int32)
    counts = torch.tensor(counts, dtype=torch.int32)
    path = torch.where(at < counts[:, None], at, -1)
    gen.keep_path(torch.arange(n).expand(len(counts), n) + 5, path, counts)


def test_a_fork_after_kept_drafts_has_all_of_them(moved):
    """Pages of what the sequence holds now, not of what the host counted before."""
    gen = generator()
    begin(gen, 0, 5, 40)
    keep(gen, [5, 0])
    assert gen.lens.tolist() == [10, 0]
    gen.fork(0, 1, 40)
    assert gen.lens.tolist() == [10, 10] and gen.counts == [10, 10]
    assert gen.pool.owned[1][:2] == gen.pool.owned[0][:2]  # two full pages
    assert moved[-1] == ("copy", [gen.pool.owned[0][2]], [gen.pool.owned[1][2]])
    assert gen.history[1, :10].tolist() == gen.history[0, :10].tolist()


def step(gen):
    """What a step does to the lengths."""
    gen._take_room()
    gen.lens += gen.live


def test_a_step_after_kept_drafts_looks_for_room(moved):
    """Where the most that drafts can have added leaves none, what they did add counts."""
    gen = generator()
    begin(gen, 0, 5, 8)
    keep(gen, [3, 0])
    with pytest.raises(ValueError):  # 8 of 8
        step(gen)
    gen.release(0)
    begin(gen, 1, 3, 8)
    keep(gen, [0, 2], 8)
    for _ in range(3):
        step(gen)
    with pytest.raises(ValueError):
        step(gen)
    assert gen.lens.tolist() == gen.counts == [0, 8]


def test_sequences_that_take_no_part_keep_their_counts(moved):
    gen = generator()
    begin(gen, 0, 5, 20)
    begin(gen, 1, 7, 20)
    gen.live[1] = False
    keep(gen, [3, 3])
    gen._count()
    assert gen.lens.tolist() == gen.counts == [8, 7]


def test_kept_drafts_stay_within_the_longest_length(moved):
    """max_len is no multiple of the page: pages have places behind it, the history has not."""
    gen = generator(2, 10, 4)
    begin(gen, 0, 5, 10)  # 12 places
    begin(gen, 1, 10, 10)
    keep(gen, [7, 3])
    assert gen.lens.tolist() == [10, 10]
    assert moved[-1][-1].tolist() == [5, 0]
    assert gen.history[0].tolist() == [0, 1, 2, 3, 4, 5, 6, 7, 8, 9]
    assert gen.history[1].tolist() == list(range(10))


def test_drafts_without_room_are_refused(moved):
    """Before anything runs: in the sequence's pages, and within the longest length."""
    gen = generator(2, 10, 4)
    node = torch.arange(4, dtype=torch.int32)
    tree = (torch.zeros(2, 4, dtype=torch.int64), node - 1, None, node)
    for tokens, room in ((5, 8), (7, 10)):
        begin(gen, 1, tokens, room)
        with pytest.raises(ValueError):
            gen.step_drafts(*tree)
        assert gen.live.tolist() == [False, True]
        gen.release(1)
    begin(gen, 1, 3, 8)
    keep(gen, [0, 2])
    with pytest.raises(ValueError):
        gen.step_drafts(*tree)


def test_generated_sequences_end_alike(moved, monkeypatch):
    """Whichever of them had its tokens first: each holds its tokens but the last and goes
    on; one that ended before does not."""
    from cuda_transformer_b200 import generate_case

    gen = generator(4, 48, 4)

    def prompts(prompts, room):
        for b, t in enumerate(prompts):
            begin(gen, b, t.numel(), t.numel() + room)
        return torch.zeros(4, 10)

    # what is found a step: 5 tokens at once, one by one, none after two, none at all
    found = [[[1], [1], [1], [-1]],
             [[2, 3, 4, 5, 6], [2, -1, -1, -1, -1], [2, -1, -1, -1, -1], [9, 9, 9, 9, 9]],
             [[9] * 5, [3] + [-1] * 4, [-1] * 5, [9] * 5]]
    kept = [[1, 1, 1, 1], [5, 1, 1, 5], [5, 1, 1, 5]]
    steps = iter(zip(found, kept))

    def verify(target, tokens, *a, **kw):
        new, counts = next(steps)
        n = tokens.shape[1]
        at = torch.arange(n, dtype=torch.int32)
        counts = torch.tensor(counts, dtype=torch.int32)
        return (torch.tensor(new)[:, :n], torch.where(at < counts[:, None], at, -1), counts)

    monkeypatch.setattr(gen, "_prompts", prompts)
    monkeypatch.setattr(gen, "_step_drafts", lambda *a: torch.zeros(4, 5, 10))
    monkeypatch.setattr(generate_case.ops, "verify_drafts", verify)
    tokens, steps = gen.generate_drafted([torch.zeros(n) for n in (3, 4, 5, 6)], 3, 4)
    assert tokens.tolist() == [[1, 2, 3], [1, 2, 3], [1, 2, -1], [-1, -1, -1]] and steps == 2
    assert gen.live.tolist() == [True, True, False, False]
    assert gen.lens.tolist() == gen.counts == [5, 6, 7, 6]
    step(gen)
    gen._count()
    assert gen.lens.tolist() == [6, 7, 7, 6]


@pytest.mark.parametrize("depth,branches", [(0, 1), (0, 3), (4, 0)])
def test_generation_with_drafts_of_no_tokens(moved, monkeypatch, depth, branches):
    """A tree of its root alone is a step of one token; fewer than none are refused."""
    from cuda_transformer_b200 import generate_case

    gen = generator()

    def prompts(prompts, room):
        for b, t in enumerate(prompts):
            begin(gen, b, t.numel(), t.numel() + room)
        return torch.zeros(2, 10)

    def verify(target, tokens, *a, **kw):
        assert tokens.shape == (2, 1)
        ones = torch.ones(2, dtype=torch.int32)
        return tokens + 1, torch.zeros(2, 1, dtype=torch.int32), ones

    def step(tokens, parents, mask, depths):
        assert parents.tolist() == [[-1]] * 2 and mask.tolist() == [[[1]]] * 2
        assert depths.tolist() == [0]
        return torch.zeros(2, 1, 10)

    monkeypatch.setattr(gen, "_prompts", prompts)
    monkeypatch.setattr(gen, "_step_drafts", step)
    monkeypatch.setattr(generate_case.ops, "verify_drafts", verify)
    some = [torch.zeros(3), torch.zeros(4)]
    tokens, steps = gen.generate_drafted(some, 3, depth, branches)
    assert tokens.tolist() == [[1, 2, 3]] * 2 and steps == 2
    for bad in ((-1, 2), (2, -1)):
        with pytest.raises(ValueError):
            gen.generate_drafted(some, 3, *bad)
