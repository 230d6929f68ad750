"""Generation with drafts and forks (cuda_transformer_b200/generate_case.py)
against running every whole sequence through the model."""
import pytest
import torch

from .test_gpu_generate import setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("cache", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("depth,branches", [(4, 1), (3, 2), (1, 5)])
def test_drafted_tokens_are_the_best_ones(cuda_device, rotary, cache, depth, branches):
    """Every token is the whole sequence's best one, up to the differences that the cache's
    type makes to the logits (twice the bounds that one-token steps are held to)."""
    from cuda_transformer_b200.generate_case import whole_sequence_logits

    model, prompts, gen = setup(cache=cache, rotary=rotary)
    tokens, steps = gen.generate_drafted(prompts, 24, depth, branches)
    assert tokens.shape == (3, 24) and 1 <= steps <= 23
    bound = 2 * {torch.float32: 2e-5, torch.bfloat16: 2e-2, torch.float16: 3e-3}[cache]
    for b, p in enumerate(prompts):
        seq = torch.cat([p, tokens[b]])
        for t in range(24):
            ref = whole_sequence_logits(model, seq[:p.numel() + t], rotary)
            assert (ref.max() - ref[tokens[b, t]]).item() <= bound, (b, t)
    # the history is what was generated, and the cache goes on from there: one more step
    n = [p.numel() + 24 for p in prompts]
    assert all(gen.lens[b] >= n[b] - 1 for b in range(3))
    for b, p in enumerate(prompts):
        have = gen.history[b, :n[b] - 1]
        assert torch.equal(have, torch.cat([p, tokens[b]])[:n[b] - 1])


def test_kept_paths_leave_the_cache_as_single_steps_do(cuda_device):
    """After drafted steps the cached keys and values of all kept tokens are those that
    one-token steps over the same tokens give (FP32; sums in another order)."""
    model, prompts, gen = setup(rotary=True)
    tokens, _ = gen.generate_drafted(prompts, 20, 3, 2)
    _, _, plain = setup(rotary=True)
    for b, p in enumerate(prompts):
        plain.prompt(b, p, p.numel() + 24)
    for t in range(19):
        plain.step(tokens[:, t])
    for (k1, v1), (k2, v2) in zip(gen.caches, plain.caches):
        for b, p in enumerate(prompts):
            at = torch.arange(p.numel() + 19, device="cuda")
            for x, y in ((k1, k2), (v1, v2)):
                one = x[gen.pool.table[b, at // 7].long(), :, at % 7]
                two = y[plain.pool.table[b, at // 7].long(), :, at % 7]
                assert (one - two).abs().max().item() <= 2e-5


def test_temperature_draws_by_the_seed(cuda_device):
    got = []
    for seed in (1, 1, 2):
        _, prompts, gen = setup()
        got.append(gen.generate_drafted(prompts, 16, 3, 2, temperature=1.0, seed=seed)[0])
    assert torch.equal(got[0], got[1]) and not torch.equal(got[0], got[2])
    assert (got[0] >= 0).all() and (got[0] < 65).all()


def test_drafts_need_room(cuda_device):
    _, prompts, gen = setup()
    with pytest.raises(ValueError):
        gen.generate_drafted(prompts, 41, 4, 1)  # 20 + 41 + 5 tokens of 64


def test_forks_go_their_own_ways(cuda_device):
    """A prompt that is given several times is run once: the same tokens as prompts run one
    by one; forks that go on differently leave each other's caches alone."""
    model, prompts, gen = setup()
    p = prompts[1]
    tokens, logits = gen.generate([p, p, p], 12)
    assert gen.pool.table[0, :2].tolist() == gen.pool.table[1, :2].tolist()  # 14 of 20 tokens
    _, _, fresh = setup()
    want, ref = fresh.generate([p, p.clone(), p.clone()], 12)
    assert torch.equal(tokens, want) and torch.equal(logits, ref)
    kw = dict(temperature=1.0, seed=3)
    one = gen.generate([p, p, p], 12, **kw)[0]
    two = fresh.generate([p, p.clone(), p.clone()], 12, **kw)[0]
    assert torch.equal(one, two) and not torch.equal(one[0], one[1])
    # a fork in the middle of a sequence
    gen.generate(prompts[:1] * 3, 10)
    gen.release(2)
    gen.fork(0, 2, 40)
    a, b = gen.step(torch.tensor([5, 7, 5], device="cuda"))[[0, 2]]
    assert torch.equal(a, b)
    gen.step(torch.tensor([1, 2, 3], device="cuda"))
    from cuda_transformer_b200.generate_case import whole_sequence_logits
    got = gen.step(torch.tensor([9, 9, 9], device="cuda"))
    for seq in (0, 2):
        n = int(gen.lens[seq])
        ref = whole_sequence_logits(model, gen.history[seq, :n])
        assert (got[seq] - ref).abs().max().item() <= 2e-5


def test_commands(cuda_device, capsys, monkeypatch):
    import json
    import sys

    from cuda_transformer_b200 import generate_case
    for extra in (["--samples", "2", "--temperature", "1"],
                  ["--drafts", "3", "--branches", "2", "--check", "--rotary"],
                  ["--drafts", "2", "--samples", "4", "--cache", "bf16", "--temperature", "0.7"]):
        argv = ["--layers", "1", "--d", "128", "--heads", "2", "--ctx", "64", "--batch", "4",
                "--new", "12"] + extra
        monkeypatch.setattr(sys, "argv", ["generate_case"] + argv)
        generate_case.main()
        line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
        assert line["value"] > 0 and line.get("below_best_logit", 0.0) <= 4e-5


def test_a_negative_root_ends_its_sequence(cuda_device):
    """Its history, its length and its cache stay as they were; the others go on."""
    _, prompts, gen = setup()
    for b, p in enumerate(prompts):
        gen.prompt(b, p, p.numel() + 8)
    before, history = gen.lens.clone(), gen.history.clone()
    tokens = torch.tensor([[1, 2], [-1, 2], [3, 4]], device="cuda")
    node = torch.arange(2, dtype=torch.int32, device="cuda")
    parents = (node - 1).expand(3, 2)
    mask = (2 ** (node + 1) - 1).int()[None, :, None].expand(3, 2, 1)
    caches = [c.clone() for pair in gen.caches for c in pair]
    gen.step_drafts(tokens, parents, mask, node)
    path = node.expand(3, 2).contiguous()
    gen.keep_path(tokens, path, torch.tensor([2, 1, 1], dtype=torch.int32, device="cuda"))
    assert gen.live.tolist() == [True, False, True]
    assert (gen.lens - before).tolist() == [2, 0, 1]
    assert torch.equal(gen.history[1], history[1])
    pages = gen.pool.owned[1]
    for c, old in zip([c for pair in gen.caches for c in pair], caches):
        assert torch.equal(c[pages], old[pages])
