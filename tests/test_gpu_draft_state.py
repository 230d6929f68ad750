"""Drafted steps, single steps and forks of the same sequences, mixed: every logit is that of
the whole sequence."""
import pytest
import torch

from .test_gpu_generate import setup

pytestmark = pytest.mark.gpu


def chain(batch, n):
    """Parents, mask and depths of chains of n nodes."""
    node = torch.arange(n, dtype=torch.int32, device="cuda")
    mask = (2 ** (node + 1) - 1).int()[None, :, None].expand(batch, n, 1)
    return (node - 1).expand(batch, n), mask, node


def path_of(counts, n):
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
    return torch.where(at < counts[:, None], at, -1), counts


def whole(model, gen, seq, rotary):
    from cuda_transformer_b200.generate_case import whole_sequence_logits

    return whole_sequence_logits(model, gen.history[seq, :int(gen.lens[seq])], rotary)


@pytest.mark.parametrize("rotary", [False, True])
def test_a_fork_after_kept_drafts(cuda_device, rotary):
    """Drafts are kept across a page's border; a fork has all of them, and both go on."""
    model, prompts, gen = setup(rotary=rotary)
    p = prompts[0]
    gen.prompt(0, p, p.numel() + 24)
    tokens = (torch.arange(10, device="cuda") * 7 % 65).expand(3, 10)
    gen.step_drafts(tokens, *chain(3, 10))
    gen.keep_path(tokens, *path_of([9, 0, 0], 10))
    gen.fork(0, 2, p.numel() + 24)
    assert gen.counts[0] == gen.counts[2] == int(gen.lens[2]) == p.numel() + 9
    for idx in ([3, -1, 4], [5, -1, 6]):
        logits = gen.step(torch.tensor(idx, device="cuda"))
        for seq in (0, 2):
            assert (logits[seq] - whole(model, gen, seq, rotary)).abs().max().item() <= 2e-5


@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("depth,branches", [(4, 1), (3, 2)])
def test_going_on_after_drafted_generation(cuda_device, rotary, depth, branches):
    """The last tokens are fed next, then others; a fork goes on as well.  Sequences that
    had all of their tokens earlier than others are among them."""
    model, prompts, gen = setup(rotary=rotary)
    tokens, _ = gen.generate_drafted(prompts, 16, depth, branches)
    assert gen.live.all()
    for b, p in enumerate(prompts):
        assert gen.history[b, :int(gen.lens[b])].tolist() == p.tolist() + tokens[b, :-1].tolist()
    for idx in (tokens[:, -1], torch.tensor([5, 9, 2], device="cuda")):
        logits = gen.step(idx)
        for seq in range(3):
            assert (logits[seq] - whole(model, gen, seq, rotary)).abs().max().item() <= 2e-5
    gen.fork(1, 0, 45)
    logits = gen.step(torch.tensor([8, 7, 6], device="cuda"))
    for seq in range(3):
        assert (logits[seq] - whole(model, gen, seq, rotary)).abs().max().item() <= 2e-5


@pytest.mark.parametrize("temperature", [0.0, 1.0, 1e-39])
def test_an_infinite_logit_is_drawn(cuda_device, temperature):
    """As in steps of one token; a temperature that makes logits infinite likewise."""
    model, prompts, gen = setup()
    if temperature < 1e-30:
        with torch.no_grad():
            model.lm_head_bias[7] = 100.0
    else:
        with torch.no_grad():
            model.lm_head_bias[7] = torch.inf
    tokens, _ = gen.generate_drafted(prompts, 6, 2, 2, temperature=temperature)
    if temperature == 1e-39:  # (1 / 1e-39 is beyond FP32: all positive logits are bounded, and drawn alike)
        from cuda_transformer_b200.generate_case import whole_sequence_logits

        for b, p in enumerate(prompts):
            seq = torch.cat([p, tokens[b]])
            for t in range(6):
                ref = whole_sequence_logits(model, seq[:p.numel() + t])
                assert tokens[b, t] >= 0 and ref[tokens[b, t]] > 0
    else:
        assert (tokens == 7).all()


def test_captured_drafted_steps(cuda_device):
    """A graph's drafted steps go unseen by the host: a fork and a step read the lengths."""
    model, prompts, gen = setup()
    for b in (0, 2):
        gen.prompt(b, prompts[b], prompts[b].numel() + 30)
    tokens = (torch.arange(12, device="cuda") * 5 % 65).view(3, 4)
    path, counts = path_of([4, 0, 2], 4)

    def drafted():
        logits = gen.step_drafts(tokens, *chain(3, 4))
        gen.keep_path(tokens, path, counts)
        return logits

    drafted()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = drafted()
    for _ in range(3):
        graph.replay()
    for b, row in ((0, 3), (2, 1)):
        assert (logits[b, row] - whole(model, gen, b, False)).abs().max().item() <= 2e-5
    gen.fork(0, 1, 24)
    assert gen.counts == gen.lens.tolist() == [17, 17, 17]
    for _ in range(7):
        out = gen.step(torch.tensor([3, 4, 5], device="cuda"))
        for b in range(3):
            assert (out[b] - whole(model, gen, b, False)).abs().max().item() <= 2e-5
    with pytest.raises(ValueError):  # the fork's 24
        gen.release(0)
        for _ in range(8):
            gen.step(torch.tensor([3, 4, 5], device="cuda"))
