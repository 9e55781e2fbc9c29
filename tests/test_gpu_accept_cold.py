"""Verification of drafted tokens at temperatures near zero, f32 logits a few steps apart, against the rule in 64 bits: a distribution that is nearly greedy is
still one, and what is far below the largest logit weighs nothing."""
import pytest

from test_gpu_accept import rule, run, spec  # noqa: F401  (the fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafted", [False, True])
@pytest.mark.parametrize("top,heat", [(10.0, 1e-9), (-3.0, 1e-8), (100.0, 1e-8), (9000.0, 1e-6), (10.0, 1e-6), (10.0, 2e-6), (1.0, 1e-7), (25.0, 1e-3)])
def test_logits_a_few_steps_apart(spec, top, heat, drafted):  # noqa: F811
    vocab, lens = 1003, [1, 4, 2, 3, 1, 2]
    rows = sum(lens)
    gen = torch.Generator().manual_seed(7)
    step = torch.nextafter(torch.tensor(top), torch.tensor(float("inf"))) - top
    target = (top - abs(float(step)) * torch.randint(0, 40, (rows, vocab), generator=gen).float()).float()
    target[::3, ::2] = -float("inf")
    tokens = target.argmax(-1).roll(1).int()  # mostly kept
    draft = torch.softmax(torch.randn(rows, vocab, generator=gen), -1) if drafted else None
    u = 0.05 + 0.9 * torch.rand(rows, generator=gen)
    args = [None if t is None else t.cuda() for t in (tokens, target, u, draft, torch.full((len(lens),), heat))]
    assert run(spec, lens, *args[:3], False, *args[3:]) == rule(lens, *args[:3], False, *args[3:])
