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
