"""The host side of forks and of drafted generation: CPU tests."""
import random

import pytest
import torch


def check_pool(pool, pages):
    held = [p for row in pool.owned for p in row]
    for b, row in enumerate(pool.owned):
        assert pool.table[b].tolist() == row + [-1] * (pool.max_pages - len(row))
        assert len(set(row)) == len(row)
    assert sorted(set(held) | set(pool.free)) == list(range(pages))
    assert not set(held) & set(pool.free) and len(set(pool.free)) == len(pool.free)
    assert all(pool.users[p] == held.count(p) for p in range(pages))


def test_forks_share_full_pages():
    """Full pages are shared, the last one is the fork's own; a page is free again when
    the last of its sequences is released."""
    from cuda_transformer_b200.generate_case import PagePool

    pool = PagePool(8, 4, 3, 6, "cpu")
    pool.reserve(0, 14)  # 4 pages, of which 10 tokens fill 2 and a half
    pairs = pool.fork(0, 1, 10)
    assert pool.owned[1][:2] == pool.owned[0][:2]
    assert pairs == [(pool.owned[0][2], pool.owned[1][2])] and pairs[0][0] != pairs[0][1]
    assert pool.fork(0, 2, 8) == [] and pool.owned[2] == pool.owned[0][:2]
    check_pool(pool, 8)
    with pytest.raises(ValueError):
        pool.fork(0, 1, 4)   # has pages
    pool.release(0)
    check_pool(pool, 8)
    pool.reserve(0, 12)
    check_pool(pool, 8)
    pool.release(2)
    with pytest.raises(ValueError):
        pool.fork(0, 2, 13)  # more tokens than pages hold
    pool.reserve(1, 20)
    with pytest.raises(RuntimeError):
        pool.fork(0, 2, 2)   # no page left for the one to copy
    assert pool.owned[2] == []
    check_pool(pool, 8)


def test_forks_at_random():
    from cuda_transformer_b200.generate_case import PagePool

    rng = random.Random(2)
    pool = PagePool(30, 3, 5, 9, "cpu")
    for _ in range(600):
        seq, other = rng.sample(range(5), 2)
        try:
            what = rng.random()
            if what < 0.3:
                pool.release(seq)
            elif what < 0.6:
                pool.reserve(seq, rng.randrange(1, 28))
            else:
                pool.fork(other, seq, rng.randrange(0, 28))
        except (RuntimeError, ValueError):
            pass
        check_pool(pool, 30)


def generator(batch=2, max_len=12, page=3):
    from cuda_transformer_b200.generate_case import Generator
    from cuda_transformer_b200.gpt_case import GPT

    return Generator(GPT(1, 64, 2, max_len, 10), batch, max_len, page)


def test_drafts_are_looked_up():
    """What followed the last token where it came up before: places after the same token
    first, later ones first; -1 where the history ends."""
    gen = generator(3)
    rows = [[1, 2, 3, 1, 2, 4, 1, 2], [5, 6, 5, 7, 5, 8, 9], [1, 1]]
    for b, row in enumerate(rows):
        gen.history[b, :len(row)] = torch.tensor(row)
        gen.lens[b] = len(row)
    # sequence 0: the root 1 comes after a 2 here and never did before: the last 1
    root = torch.tensor([1, 5, 3])
    got = gen.look_up_drafts(root, 3, 2)
    assert got[0].tolist() == [1, 2, -1, -1, 2, 4, 1]
    assert got[1].tolist() == [5, 8, 9, -1, 7, 5, 8]
    assert got[2].tolist() == [3] + [-1] * 6
    gen.history[0, :8] = torch.tensor([7, 1, 5, 5, 1, 6, 6, 7])  # 7 1 before, and 1 later
    assert gen.look_up_drafts(root, 2, 2)[0].tolist() == [1, 5, 5, 6, 6]
    assert gen.look_up_drafts(torch.tensor([-1, -1, -1]), 2, 1).tolist() == [[-1, -1, -1]] * 3


def test_forks_are_checked():
    gen = generator()
    with pytest.raises(ValueError):
        gen.fork(0, 1)
    gen.pool.reserve(0, 4)
    gen.counts[0] = 4
    for dst, room in ((0, 0), (1, 13)):
        with pytest.raises(ValueError):
            gen.fork(0, dst, room)
    with pytest.raises(ValueError):
        gen.generate_drafted([torch.zeros(1, dtype=torch.int64)], 4)


def test_a_fork_without_room_leaves_nothing_behind():
    gen = generator(2, 12, 3)
    gen.pool.reserve(0, 12)
    gen.counts[0] = 4
    while len(gen.pool.free) > 1:  # (one page: for the copy, not for more)
        gen.pool.free.pop()
    with pytest.raises(RuntimeError):
        gen.fork(0, 1, 12)
    assert gen.pool.owned[1] == [] and len(gen.pool.free) == 1 and gen.counts[1] == 0
    assert gen.pool.users[gen.pool.owned[0][0]] == 1
