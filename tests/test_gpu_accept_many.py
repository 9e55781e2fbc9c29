"""Verification of drafted tokens for as many requests as a busy server has: the launch forms of more than a handful of requests (clusters of eight blocks of sixteen
warps, and of eight) against the rule in 64 bits, token for token, and against the same requests by themselves."""
import pytest

from test_gpu_accept import case, rule, run, spec  # noqa: F401  (the fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["probs", "bf16", "f32"])
@pytest.mark.parametrize("drafted,greedy", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("requests,vocab,pad", [(8, 50001, 0), (12, 50001, 0), (17, 32768, 3), (40, 50001, 0), (90, 5003, 1)])
def test_equal_to_the_rule(spec, kind, drafted, greedy, requests, vocab, pad):  # noqa: F811
    lens = [(5 * i * i + 3 * i) % 9 for i in range(requests)]
    lens[1] = 11  # more rows than are judged at a time
    tokens, target, u, draft, temperature = case(lens, vocab, kind, drafted, greedy, requests, pad)
    if kind != "probs":  # mostly kept, so that windows are read to their end
        first = 0
        for b, n in enumerate(lens):
            if n > 1 and b % 3:
                tokens[first + 1:first + n] = target[first:first + n - 1].float().argmax(-1).int()
            first += n
    assert run(spec, lens, tokens, target, u, kind == "probs", draft, temperature) == rule(lens, tokens, target, u, kind == "probs", draft, temperature)


def test_every_request_greedy(spec):  # noqa: F811
    lens, vocab = [8 - i % 4 for i in range(48)], 131072
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows = sum(lens)
    target = (torch.randn(rows, vocab, generator=gen, device="cuda") * 3).bfloat16()
    best = target.float().argmax(-1).int()
    tokens = best.roll(1)
    off = torch.rand(rows, generator=gen, device="cuda") < 0.1
    tokens[off] = torch.randint(0, vocab, (int(off.sum()),), dtype=torch.int32, generator=gen, device="cuda")
    heat, u = torch.zeros(len(lens), device="cuda"), torch.rand(rows, generator=gen, device="cuda")
    assert run(spec, lens, tokens, target, u, False, None, heat) == rule(lens, tokens, target, u, False, None, heat)


@pytest.mark.parametrize("kind", ["probs", "f32"])
def test_the_same_requests_by_themselves(spec, kind):  # noqa: F811
    """Another launch form adds in another order: its sums move by 1e-7 and 1e-15, which these numbers are not that near to."""
    lens = [4] * 40
    tokens, target, u, draft, _ = case(lens, 20011, kind, True, False, 5)
    together = run(spec, lens, tokens, target, u, kind == "probs", draft)
    for b in range(0, 40, 7):
        part = slice(4 * b, 4 * b + 4)
        alone = run(spec, [4], tokens[part].contiguous(), target[part], u[part].contiguous(), kind == "probs", draft[part])
        assert alone == ([together[0][b]], [together[1][b]])
