"""The example model (``kdn_b200.decoder``): training and generation on the package's operators together.

Tolerance of the logits: the whole-sequence path rounds to bf16 after every
operator (about ten roundings of 2^-9 per layer on the way to the logits, two
layers), the token path rounds less: 5e-2 of the largest logit.
"""
import pytest
import torch

from kdn_b200.decoder import KDNDecoder

VOCAB, HEADS = 257, 2


def make(variant, seed=0, **kw):
    torch.manual_seed(seed)
    return KDNDecoder(VOCAB, 192, 2, HEADS, variant=variant, inner=320, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
@pytest.mark.parametrize("kw", [{}, {"post_norm": True, "scale_init": 0.5, "stream": torch.bfloat16}])
def test_tokens_one_by_one_agree_with_the_whole_sequence(variant, kw):
    model = make(variant, **kw)
    tokens = torch.randint(VOCAB, (3, 80), device="cuda")
    with torch.no_grad():
        whole = model(tokens).float()
    pools, steps = model.make_pools(5), [m.make_step() for m in model.mixers]
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    at = 66  # the prompt ends inside a chunk
    logits = [model.start(tokens[:, :at], pools, slots.long())]
    logits += [model.decode(tokens[:, t], pools, steps, slots) for t in range(at, 80)]
    got = torch.stack(logits, 1).float()
    want = whole[:, at - 1:]
    assert (got - want).abs().max() < 5e-2 * want.abs().max()
    for pool in pools:  # slots that are not in the call stay empty
        assert (pool.memory[[1, 3]] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_generation_repeats_and_the_graph_changes_nothing(variant):
    model = make(variant, seed=1)
    prompts = torch.randint(VOCAB, (4, 5), device="cuda")
    outs = []
    for graph in (True, True, False):
        gen = torch.Generator(device="cuda").manual_seed(3)
        outs.append(model.generate(prompts, 12, generator=gen, graph=graph, temperature=0.9, top_k=40, top_p=0.9,
                                   min_p=0.01))
    for tokens, probs in outs:
        assert tokens.shape == probs.shape == (4, 12) and tokens.min() >= 0 and tokens.max() < VOCAB
        assert torch.equal(tokens, outs[0][0]) and torch.equal(probs, outs[0][1])
    greedy, _ = model.generate(prompts, 3, temperature=0.0)
    with torch.no_grad():
        assert torch.equal(greedy[:, 0], model(prompts)[:, -1].float().argmax(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_trains(variant):
    """Ten optimizer steps on one batch: every parameter gets a finite gradient and the loss falls by a third."""
    model = make(variant, seed=2, post_norm=True, scale_init=1.0)
    tokens = torch.randint(VOCAB, (2, 65), device="cuda")
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(10):
        logits = model(tokens[:, :-1])
        loss = torch.nn.functional.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < losses[0] * 2 / 3, losses


def test_refuses_unknown_variants():
    with pytest.raises(ValueError, match="variant"):
        KDNDecoder(16, 128, 1, 1, variant="other", device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("variant", ["iso", "diag"])
def test_rows_without_a_token_go_on(variant):
    """Logits that are all NaN give token -1, which must not reach the embedding."""
    model = make(variant, seed=5)
    prompts = torch.randint(VOCAB, (3, 9), device="cuda")
    with torch.no_grad():
        model.head.weight.fill_(float("nan"))
    for graph in (True, False):
        tokens, probs = model.generate(prompts, 6, graph=graph, top_k=3)
        assert tokens.shape == (3, 6) and (tokens == -1).all() and (probs == 0).all()


def test_no_new_tokens_and_empty_prompts():
    model = KDNDecoder(16, 128, 1, 1, device="cpu")
    prompts = torch.zeros(3, 5, dtype=torch.int64)
    tokens, probs = model.generate(prompts, 0)
    assert tokens.shape == probs.shape == (3, 0) and tokens.dtype == torch.int64 and probs.dtype == torch.float32
    with pytest.raises(ValueError, match="count"):
        model.generate(prompts, -1)
    with pytest.raises(ValueError, match="prompts must be"):
        model.generate(prompts[:, :0], 4)
    with pytest.raises(ValueError, match="prompts must be"):
        model.generate(prompts[0], 4)


@pytest.mark.gpu
def test_one_new_token():
    model = make("iso", seed=6)
    prompts = torch.randint(VOCAB, (2, 1), device="cuda")
    tokens, probs = model.generate(prompts, 1, temperature=0.0)
    with torch.no_grad():
        assert torch.equal(tokens[:, 0], model(prompts)[:, -1].float().argmax(-1)) and (probs == 1).all()
