"""Generation over the paged cache (cuda_transformer_b200/generate_case.py)
against running every whole sequence through the model."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def setup(batch=3, cache=torch.float32, rotary=False, page=7, ctx=64, vocab=65):
    from cuda_transformer_b200.generate_case import Generator
    from cuda_transformer_b200.gpt_case import GPT

    torch.manual_seed(3)
    model = GPT(2, 128, 4, ctx, vocab).cuda()
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, vocab, (n,), generator=g).cuda() for n in (1, 20, 9)[:batch]]
    return model, prompts, Generator(model, batch, ctx, page, cache, rotary)


@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("cache", [torch.float32, torch.bfloat16, torch.float16])
def test_matches_whole_sequences(cuda_device, cache, graph, rotary):
    """Logits of every step; with an FP32 cache only the order of sums differs
    (3xTF32 products: 2^-21 of terms below 4 over a few hundred of them), a
    16-bit one rounds keys and values by 2^-9 or 2^-12 of values below 4, which
    two blocks with weights of 0.02 carry to the logits attenuated."""
    from cuda_transformer_b200.generate_case import whole_sequence_logits

    model, prompts, gen = setup(cache=cache, rotary=rotary)
    tokens, logits = gen.generate(prompts, 24, graph=graph)
    bound = {torch.float32: 2e-5, torch.bfloat16: 2e-2, torch.float16: 3e-3}[cache]
    for b, p in enumerate(prompts):
        seq = torch.cat([p, tokens[b]])
        for t in range(24):
            ref = whole_sequence_logits(model, seq[:p.numel() + t], rotary)
            assert (ref - logits[t, b]).abs().max().item() <= bound, (b, t)
            assert logits[t, b, tokens[b, t]] == logits[t, b].max()


def test_penalties_and_mask_steer_the_choice(cuda_device):
    """A presence penalty above the logits' range forbids a second use of any
    generated token; a mask keeps the choice to its tokens; a bias decides."""
    model, prompts, gen = setup()
    tokens, _ = gen.generate(prompts, 30, presence=torch.full((3,), 100.0, device="cuda"))
    assert all(row.unique().numel() == 30 for row in tokens)
    mask = torch.zeros(3, 3, dtype=torch.int32, device="cuda")
    mask[:, 1] = 0b1010  # tokens 33 and 35
    tokens, _ = gen.generate(prompts, 12, temperature=1.0, mask=mask)
    assert set(tokens.unique().tolist()) <= {33, 35}
    ids = torch.full((3, 1), 50, device="cuda")
    tokens, _ = gen.generate(prompts, 5, bias_ids=ids,
                             bias_values=torch.full((3, 1), 100.0, device="cuda"))
    assert (tokens == 50).all()


def test_graph_and_eager_choose_alike(cuda_device):
    kw = {k: torch.full((3,), x, device="cuda")
          for k, x in (("repetition", 1.2), ("frequency", 0.1), ("presence", 0.1))}
    got = []
    for graph in (False, True):
        _, prompts, gen = setup(rotary=True, cache=torch.bfloat16)
        got.append(gen.generate(prompts, 30, temperature=0.9, seed=5, graph=graph, **kw)[0])
    assert torch.equal(*got)


def test_sequences_can_be_replaced(cuda_device):
    """A released sequence's pages serve another prompt; its old values leave no trace."""
    model, prompts, gen = setup()
    gen.generate(prompts, 40)
    want = gen.generate(prompts[::-1], 10)[0]
    _, _, fresh = setup()
    assert torch.equal(want, fresh.generate(prompts[::-1], 10)[0])


def test_no_token_left(cuda_device):
    """A row whose mask leaves nothing, or whose logits are NaN, has no next token: -1, with
    and without a temperature, and it has ended: nothing more is fed to it."""
    for temperature in (0.0, 0.7):
        model, prompts, gen = setup()
        mask = torch.full((3, 3), -1, dtype=torch.int32, device="cuda")
        mask[1] = 0
        tokens, logits = gen.generate(prompts, 6, temperature=temperature, mask=mask)
        assert (tokens[1] == -1).all() and (tokens[[0, 2]] >= 0).all()
        assert gen.lens.tolist() == [p.numel() + n for p, n in zip(prompts, (6, 0, 6))]
        _, _, other = setup()
        want, ref = other.generate(prompts, 6, temperature=temperature)
        assert torch.equal(tokens[[0, 2]], want[[0, 2]])
        assert torch.equal(logits[:, [0, 2]], ref[:, [0, 2]])
        bad = ref[0].clone()
        bad[2] = float("nan")
        uniform = torch.full((3,), 0.5, device="cuda")
        got = other.choose(bad, temperature, uniform)
        assert got[2] == -1 and got[0] >= 0


def test_infinite_bias_decides(cuda_device):
    for temperature in (0.0, 0.9):
        model, prompts, gen = setup()
        tokens, _ = gen.generate(prompts, 4, temperature=temperature,
                                 bias_ids=torch.full((3, 1), 11, device="cuda"),
                                 bias_values=torch.full((3, 1), float("inf"), device="cuda"))
        assert (tokens == 11).all()


def test_a_drawn_token_has_a_probability(cuda_device):
    """The running sums of a parallel scan can step up by a rounding at a token of
    probability 0; numbers that fall into such a step must not draw it."""
    from cuda_transformer_b200.generate_case import Generator
    from cuda_transformer_b200.gpt_case import GPT

    vocab = 60000
    gen = Generator(GPT(1, 64, 2, 8, vocab).cuda(), 1, 8)
    gen.prompt(0, torch.zeros(1, dtype=torch.int64, device="cuda"), 8)
    g, steps = torch.Generator(device="cuda").manual_seed(1), 0
    from cuda_transformer import ops
    for _ in range(20):
        logits = 3 * torch.randn(1, vocab, generator=g, device="cuda")
        mask = torch.randint(-2 ** 31, 2 ** 31, (1, vocab // 32), generator=g, device="cuda").int()
        masked = ops.logits_process(logits, mask=mask)
        probs = ops.cuda_softmax(masked.unsqueeze(0))[0]
        upto = probs.cumsum(-1)[0]
        rises = ((probs[0, 1:] == 0) & (upto[1:] > upto[:-1])).nonzero()[:8, 0] + 1
        for i in rises.tolist():
            uniform = (upto[i - 1] / upto[-1])[None].clamp(max=1 - 2.0 ** -24)
            idx = gen.choose(logits, 1.0, uniform, mask=mask)
            assert probs[0, idx] > 0
            steps += 1
    print("steps at tokens of probability 0:", steps)
