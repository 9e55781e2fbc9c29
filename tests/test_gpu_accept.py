"""Verification of drafted tokens against the rule, row by row, in 64 bits.  Whole numbers: everything has to be equal."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def spec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return importlib.import_module("glm53f-afd_b200.spec")


def rule(lens, tokens, target, u, probabilities, draft, temperature):
    """The definition, on the host."""
    target, u = target.cpu().double(), u.cpu().double()
    draft = None if draft is None else draft.cpu().double()
    tokens, vocab = tokens.tolist(), target.shape[1]
    keeps, nexts = [], []
    first = 0
    for b, n in enumerate(lens):
        if n == 0:
            keeps.append(0), nexts.append(-1)
            continue
        heat = None if probabilities else 1.0 if temperature is None else float(temperature[b])

        def p_of(i):
            row = target[first + i]
            if probabilities:
                return torch.where((row > 0) & (row < math.inf), row, 0.0)
            row = torch.where(row.isnan(), -math.inf, row)
            top = row.max()
            if top == -math.inf:
                return torch.zeros(vocab, dtype=torch.float64)
            e = torch.where(row == top, 1.0, torch.exp((row - top) / heat))
            return e / e.sum()

        def best_of(i):
            row = torch.where(target[first + i].isnan(), -math.inf, target[first + i])
            return -1 if row.max() == -math.inf else int((row == row.max()).nonzero()[0])

        kept = 1
        while kept < n:
            t = tokens[first + kept]
            if heat is not None and heat <= 0:
                ok = t >= 0 and t == best_of(kept - 1)
            elif not 0 <= t < vocab:
                ok = False
            else:
                ok = float(u[first + kept]) * (1.0 if draft is None else float(draft[first + kept, t])) < float(p_of(kept - 1)[t])
            if not ok:
                break
            kept += 1
        if heat is not None and heat <= 0:
            nexts.append(best_of(kept - 1))
        else:
            w = p_of(kept - 1)
            if kept < n:
                t = tokens[first + kept]
                less = w.clone() if draft is None else (w - draft[first + kept]).clamp(min=0)
                if draft is None and 0 <= t < vocab:
                    less[t] = 0
                w = less if float(less.sum()) > 0 else w
            if float(w.sum()) > 0:
                upto = w.cumsum(0)
                at = int((upto <= float(u[first]) * float(upto[-1])).sum())
                nexts.append(at if at < vocab else int(w.nonzero()[-1]))
            else:
                nexts.append(-1)
        keeps.append(kept)
        first += n
    return keeps, nexts


def case(lens, vocab, kind, drafted, greedy, seed, pad=0, sharp=3.0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(lens)
    logits = sharp * torch.randn(rows, vocab, generator=gen)
    guess = torch.roll(logits, 1, 0) + 0.7 * torch.randn(rows, vocab, generator=gen)
    if drafted:
        draft = torch.softmax(guess, -1)
        tokens = torch.multinomial(draft, 1, generator=gen)[:, 0]
    else:
        draft, tokens = None, guess.argmax(-1)
    target = torch.softmax(logits, -1) if kind == "probs" else logits.to(torch.bfloat16 if kind == "bf16" else torch.float32)
    temperature = None
    if kind != "probs" and greedy:
        temperature = 0.5 + torch.rand(len(lens), generator=gen)
        temperature[::2] = 0.0
    if pad:
        wide = torch.full((rows, vocab + pad), 50.0, dtype=target.dtype)
        wide[:, :vocab] = target
        target = wide
    u = torch.rand(rows, generator=gen)
    put = lambda t: None if t is None else t.cuda()
    target = put(target)[:, :vocab] if pad else put(target)
    return tokens.int().cuda(), target, u.cuda(), put(draft), put(temperature)


def run(spec, lens, tokens, target, u, probabilities=False, draft=None, temperature=None):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    keep, nxt = (torch.full((len(lens) + 1,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    spec.accept_batch(torch.tensor(cu, dtype=torch.int32, device="cuda"), tokens, target, u, keep, nxt, probabilities=probabilities, draft=draft,
                      temperature=temperature)
    torch.cuda.synchronize()
    assert keep[-1] == -7 and nxt[-1] == -7
    return keep[:-1].tolist(), nxt[:-1].tolist()


@pytest.mark.parametrize("kind", ["probs", "bf16", "f32"])
@pytest.mark.parametrize("drafted,greedy", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("lens,vocab,pad", [([8], 32768, 0), ([1, 3, 0, 8, 2, 20, 9], 1003, 5), ([2, 5, 4], 1, 0), ([4, 4, 1, 6], 37, 3), ([3, 8, 7, 2], 50001, 0)])
def test_equal_to_the_rule(spec, kind, drafted, greedy, lens, vocab, pad):
    for seed in range(3):
        tokens, target, u, draft, temperature = case(lens, vocab, kind, drafted, greedy, seed, pad)
        got = run(spec, lens, tokens, target, u, kind == "probs", draft, temperature)
        assert got == rule(lens, tokens, target, u, kind == "probs", draft, temperature)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_masked_rows_ties_and_bad_tokens(spec, kind):
    lens, vocab = [3, 3, 2, 2, 2, 1, 2], 300
    tokens, target, u, _, _ = case(lens, vocab, kind, False, False, 4)
    inf = float("inf")
    target[0, :] = -inf          # a row that leaves nothing
    target[3, 10:200] = -inf     # masked entries, the rest drawn from
    target[4, 5] = float("nan")
    target[6, 17] = target[6, 250] = inf   # the two share everything
    target[8, :] = 2.0           # all equal
    target[10, :] = float("nan")
    target[11, :] = torch.finfo(target.dtype).min
    tokens[1], tokens[4], tokens[7], tokens[9] = 0, 20, 17, vocab   # tokens[4] is masked in row 3, tokens[9] is none
    tokens[12 + 1] = -3
    for temperature in (None, torch.tensor([0.0, 1.0, 0.0, 2.0, 0.0, 1.0, 0.0], device="cuda"), torch.zeros(7, device="cuda")):
        assert run(spec, lens, tokens, target, u, False, None, temperature) == rule(lens, tokens, target, u, False, None, temperature)


def test_random_numbers_at_their_ends(spec):
    lens, vocab = [2, 2, 2, 1, 1], 4097
    tokens, target, u, draft, _ = case(lens, vocab, "probs", True, False, 6)
    for first, judge in ((0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (0.0, 1 - 2.0 ** -24)):
        u[0::2], u[1::2] = first, judge
        assert run(spec, lens, tokens, target, u, True, draft) == rule(lens, tokens, target, u, True, draft, None)
    # The drafter's distribution is the target's: every token is kept; and where it is refused all the same (u = 1 is none of
    # these numbers), nothing is left of max(p - q, 0) and the draw is from p.
    draft[1] = target[0]
    draft[3] = target[2]
    u[:] = 0.5
    keep, nxt = run(spec, lens, tokens, target, u, True, draft)
    assert keep[:2] == [2, 2]
    u[1] = 1.0
    assert run(spec, lens, tokens, target, u, True, draft) == rule(lens, tokens, target, u, True, draft, None)


def test_probabilities_that_are_none(spec):
    lens, vocab = [2, 1, 2], 129
    tokens, target, u, draft, _ = case(lens, vocab, "probs", True, False, 8)
    target[2, 3:60] = -0.25
    target[2, 60] = float("nan")
    target[2, 61] = float("inf")
    target[3] = 0.0
    assert run(spec, lens, tokens, target, u, True, draft) == rule(lens, tokens, target, u, True, draft, None)


def test_frequencies_are_the_targets(spec):
    """Over many windows of one draft the first new token is distributed as the target's: 64 equal windows a call, 512 calls; every count within
    five standard deviations of its expectation (chance of one of twelve beyond: below 1e-5)."""
    vocab, windows, calls = 12, 64, 512
    gen = torch.Generator().manual_seed(1)
    p = torch.softmax(torch.randn(vocab, generator=gen), 0)
    q = torch.softmax(torch.randn(vocab, generator=gen), 0)
    target = p.log().repeat(2 * windows, 1).cuda()
    draft = q.repeat(2 * windows, 1).cuda()
    counts = torch.zeros(vocab)
    cu = torch.arange(0, 2 * windows + 1, 2, dtype=torch.int32, device="cuda")
    keep, nxt = (torch.empty(windows, dtype=torch.int32, device="cuda") for _ in range(2))
    for _ in range(calls):
        tokens = torch.multinomial(q, 2 * windows, replacement=True, generator=gen).int().cuda()
        u = torch.rand(2 * windows, generator=gen).cuda()
        spec.accept_batch(cu, tokens, target, u, keep, nxt, draft=draft)
        new = torch.where(keep == 2, tokens[1::2], nxt)
        counts += torch.bincount(new.cpu(), minlength=vocab)
    n = windows * calls
    assert bool(((counts - n * p).abs() < 5 * (n * p * (1 - p)).sqrt()).all())


def test_a_replayed_graph_reads_new_numbers(spec):
    lens, vocab = [4, 2], 5000
    tokens, target, u, draft, _ = case(lens, vocab, "f32", True, False, 10)
    cu = torch.tensor([0, 4, 6], dtype=torch.int32, device="cuda")
    keep, nxt = (torch.empty(2, dtype=torch.int32, device="cuda") for _ in range(2))
    spec.accept_batch(cu, tokens, target, u, keep, nxt, draft=draft)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spec.accept_batch(cu, tokens, target, u, keep, nxt, draft=draft)
    for seed in (11, 12, 13):
        other = case(lens, vocab, "f32", True, False, seed)
        for old, new in zip((tokens, target, u, draft), other):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert (keep.tolist(), nxt.tolist()) == rule(lens, tokens, target, u, False, draft, None)
