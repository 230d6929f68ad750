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
