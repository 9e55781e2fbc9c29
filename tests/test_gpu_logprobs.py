"""Log probabilities, entropy, alternatives and their gradients on the GPU against 64 bits.

Bounds, u = 2^-24.  (x - max) log2(e) / T is formed to 4 u of itself, each power of two to 4 u, and a lane adds at most vocab / 512 + 150 numbers one after another, rescalings
counted as ten additions each (at most one for 8,192 values, and a dozen where sums meet): S, and the sum behind the entropy, are within s = u (vocab / 512 + 150) + 4 u |t| of
themselves for the terms' |t|, of which those above 30 are below e^-30 of the sum: s = u (vocab / 512 + 300)."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24
INF, NAN = math.inf, math.nan


@pytest.fixture(scope="module")
def spec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.spec")


def heat_of(temperature, rows):
    if temperature is None:
        return torch.ones(rows, 1, dtype=torch.float64, device="cuda")
    t = temperature.double()
    return torch.where(t > 0, t.clamp(1e-30, 1e30), 1.0)[:, None]  # (a NaN is not above 0)


def exact(logits, temperature):
    """(log p, entropy) in 64 bits; rows of which nothing is left: -inf and 0."""
    x = logits.double()
    top = x.amax(1, keepdim=True)
    t = (x - torch.where(top == -INF, 0.0, top)) / heat_of(temperature, len(x))
    logp = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    logp = torch.where(top == -INF, torch.full_like(logp, -INF), logp)
    return logp, -(torch.exp(logp) * logp.masked_fill(logp == -INF, 0.0)).sum(1)


def best_of(logits, k):
    """The k largest entries above -inf, ties to the lowest index: indices, -1 where there are no more."""
    x = logits.float()
    x = torch.where(x.isnan(), -INF, x)
    order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    order = torch.where(torch.gather(x, 1, order) == -INF, -1, order)
    return torch.nn.functional.pad(order, (0, k - order.shape[1]), value=-1)


def run(spec, logits, tokens, temperature=None, top=0):
    rows = len(logits)
    f = lambda *s: torch.full(s, 77.0, device="cuda")
    logprob, entropy, lse = f(rows), f(rows), f(rows)
    pair = (torch.full((rows, top), 77, dtype=torch.int32, device="cuda"), f(rows, top)) if top else None
    spec.logprobs(logits, tokens, logprob, temperature=temperature, entropy=entropy, lse=lse, top=pair)
    return logprob, entropy, lse, pair


def check(spec, logits, tokens, temperature=None, top=0):
    rows, vocab = logits.shape
    logprob, entropy, lse, pair = run(spec, logits, tokens, temperature, top)
    logp, h = exact(logits, temperature)
    s = U * (vocab / 512 + 300)
    token = tokens.long()
    named = (token >= 0) & (token < vocab)
    want = torch.where(named, logp.gather(1, token.clamp(0, vocab - 1)[:, None])[:, 0], 0.0)

    def near(got, want, what):
        got, same = got.double(), (got.double() == want)
        # 4 u |t| of the term's own t, that is of log p and log S, with two roundings each: 10 u of both at any size, 4.9e32 too (only infinities are compared as they are).
        tol = s + 10 * U * want.abs().masked_fill(want.isinf(), 0.0) + 10 * U * math.log(vocab + 1)
        assert (same | ((got - want).abs() <= tol)).all(), (what, (got - want).abs().nan_to_num().max())

    near(logprob, want, "logprob")
    assert ((entropy.double() - h).abs() <= 2 * s * (1 + h) + 10 * U * (h + math.log(vocab + 1))).all(), (entropy.double() - h).abs().max()
    if top:
        ids, values = pair
        order = best_of(logits, top)
        assert torch.equal(ids.long(), order)
        value = torch.where(order < 0, -INF, logp.gather(1, order.clamp(min=0)))
        near(values, value, "values")
    return logprob, entropy, lse


def make(rows, vocab, dtype, seed=1, pad=0, shift=0, span=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    room = torch.randn(rows * (vocab + pad) + shift + 8, generator=gen, device="cuda").mul_(span).to(dtype)
    return room[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab], gen


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,pad,shift,top", [
    (1, 1, 0, 0, 1), (3, 2, 0, 1, 5), (2, 7, 1, 0, 32), (5, 31, 0, 3, 20), (9, 1000, 0, 0, 32), (4, 4097, 2, 1, 20), (3, 50257, 0, 0, 5), (1, 131072, 0, 0, 20), (300, 8191, 0, 0, 1),
    (2, 262145, 3, 2, 32), (600, 260, 4, 0, 0), (1, 2000000, 0, 5, 32)])
def test_rows(spec, dtype, rows, vocab, pad, shift, top):
    logits, gen = make(rows, vocab, dtype, pad=pad, shift=shift)
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    check(spec, logits, tokens, None, top)
    temperature = 0.5 + torch.rand(rows, generator=gen, device="cuda")
    first = check(spec, logits, tokens, temperature, top)
    again = run(spec, logits, tokens, temperature, top)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [513, 20000])
def test_orders_of_the_logits(spec, dtype, vocab):
    """Ascending and descending rows, ties, constant rows, the best all in one place, huge and tiny spans."""
    line = torch.arange(vocab, device="cuda", dtype=F32)
    rows = [line * 1e-3, -line * 1e-3, torch.zeros(vocab, device="cuda"), (line % 3), (line // 600), torch.where(line > vocab - 40, 5.0, 0.0), torch.where(line < 40, 5.0, -3.0),
            line * 1e30, -line * 1e-30, torch.where(line == 17, 0.0, -INF), torch.where(line % 2 == 0, -INF, line % 7), torch.where(line % 9 == 0, -0.0, 0.0), line * 0 - 1e4]
    logits = torch.stack(rows).to(dtype)
    tokens = torch.arange(len(rows), device="cuda", dtype=torch.int32) * 3 % vocab
    for top in (1, 20, 32):
        check(spec, logits, tokens, None, top)


def test_rows_with_nothing_and_with_what_is_no_number(spec):
    vocab = 3001
    for dtype in (BF, F32):
        logits, _ = make(7, vocab, dtype)
        logits[0] = -INF
        logits[1, 1::2] = -INF
        logits[2, 100], logits[3, 5], logits[4] = NAN, INF, NAN
        logits[5, :] = -INF
        logits[5, 3000] = -7.0
        tokens = torch.tensor([3, 1, 7, 5, 0, 3000, -1], dtype=torch.int32, device="cuda")
        logprob, entropy, lse, (ids, values) = run(spec, logits, tokens, None, 4)
        assert logprob[0] == -INF and entropy[0] == 0 and lse[0] == -INF and (ids[0] == -1).all() and (values[0] == -INF).all()
        assert logprob[1] == -INF and logprob[6] == 0
        for r in (2, 3, 4):
            assert logprob[r].isnan() and entropy[r].isnan() and lse[r].isnan()
        assert torch.equal(ids.long(), best_of(logits, 4)) and ids[3, 0] == 5 and (ids[4] == -1).all() and values[2].isnan().all()
        assert logprob[5] == 0 and entropy[5] == 0 and lse[5] == -7 and ids[5].tolist() == [3000, -1, -1, -1] and values[5, 0] == 0
        d = torch.full_like(logits, 3.0)
        one = torch.ones(7, device="cuda")
        spec.logprobs_backward(logits, tokens, lse, one, d, entropy=entropy, dentropy=one)
        assert (d[0] == 0).all() and (d[1, 1::2] == 0).all() or d[1, 1] == 1  # (the token of row 1 is a masked one)
        assert d[2].isnan().all() and not d[1].isnan().any() and (d[5, :3000] == 0).all() and d[5, 3000] == 0
        clean = logits[1:2].clone()
        assert not d[6].isnan().any() and clean is not None


def test_temperatures(spec):
    logits, _ = make(9, 5000, F32)
    t = torch.tensor([0.0, -1.0, NAN, 1.0, 1e-30, 1e38, 1e-45, 0.01, 100.0], device="cuda")
    tokens = logits.argmax(1).int()
    check(spec, logits, tokens, t, 3)
    a, b = run(spec, logits, tokens, t, 3), run(spec, logits, tokens, None, 3)
    for x, y in zip((*a[:3], *a[3]), (*b[:3], *b[3])):
        assert torch.equal(x[:4], y[:4])
    assert (a[0][4:5] == 0).all()


def grads(logits, tokens, temperature, dl, dn):
    logp, h = exact(logits, temperature)
    p = logp.exp()
    l, n = ((torch.zeros(len(p), 1, dtype=torch.float64, device="cuda") if g is None else g.double()[:, None]) for g in (dl, dn))
    rows, vocab = p.shape
    named = (tokens >= 0) & (tokens < vocab)
    l = l * named[:, None]
    safe = logp.masked_fill(logp == -INF, 0.0)
    d = -l * p - n * p * (safe + h[:, None])
    d.scatter_add_(1, tokens.long().clamp(0, vocab - 1)[:, None], l)
    heat = heat_of(temperature, rows)
    # p to 8 u |log p| and the sum's s; the entropy to 2 s (1 + H)
    s = U * (vocab / 512 + 300)
    rel = s + U * (8 * safe.abs() + 20 + 4 * (logits.double().amax(1, keepdim=True) / heat).abs())
    bound = p * (l.abs() + n.abs() * (safe.abs() + h[:, None])) * rel + n.abs() * p * (4 * s * (1 + h[:, None]) + 16 * U * (safe.abs() + h[:, None]))
    bound.scatter_add_(1, tokens.long().clamp(0, vocab - 1)[:, None], 8 * U * l.abs())
    return d / heat, bound / heat + 1e-37


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,pad,shift,heat", [(1, 1, 0, 0, False), (3, 7, 2, 1, True), (4, 50257, 0, 0, False), (2, 131072, 0, 0, True), (33, 1000, 5, 3, True)])
def test_gradients(spec, dtype, rows, vocab, pad, shift, heat):
    logits, gen = make(rows, vocab, dtype, pad=pad, shift=shift)
    if vocab > 100:
        logits[:, 5::17] = -INF
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[-1:] = -100 if rows > 2 else 0
    temperature = 0.5 + torch.rand(rows, generator=gen, device="cuda") if heat else None
    _, entropy, lse, _ = run(spec, logits, tokens, temperature)
    dl, dn = torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda")
    for a, b in ((dl, dn), (dl, None), (None, dn)):
        want, bound = grads(logits, tokens, temperature, a, b)
        step = torch.finfo(dtype).eps / 2 * (want.abs() + bound)
        room = make(rows, vocab, dtype, seed=2, pad=1 if vocab < 200 else 0, shift=0)[0]
        for out in (room, torch.empty(rows, vocab, dtype=dtype, device="cuda"), logits.clone()):
            source = out if out.data_ptr() != room.data_ptr() and torch.equal(out, logits) else logits  # in place
            spec.logprobs_backward(source, tokens, lse, a, out, temperature=temperature, entropy=entropy if b is not None else None, dentropy=b)
            assert ((out.double() - want).abs() <= bound + step).all(), ((out.double() - want).abs() / (bound + step)).max()
        if pad and vocab > 1:
            assert not logits.isnan().any()


def test_gradients_against_differences(spec):
    logits, gen = make(4, 300, F32)
    tokens = torch.tensor([0, 299, 17, 5], dtype=torch.int32, device="cuda")
    t = torch.tensor([0.7, 1.0, 1.5, 2.0], device="cuda")
    _, entropy, lse, _ = run(spec, logits, tokens, t)
    dl, dn = torch.randn(4, generator=gen, device="cuda"), torch.randn(4, generator=gen, device="cuda")
    d = torch.empty_like(logits)
    spec.logprobs_backward(logits, tokens, lse, dl, d, temperature=t, entropy=entropy, dentropy=dn)
    move = torch.randn(4, 300, generator=gen, device="cuda", dtype=torch.float64)

    def loss(eps):
        logp, h = exact(logits.double() + eps * move, t)
        return float((logp.gather(1, tokens.long()[:, None])[:, 0] * dl.double() + h * dn.double()).sum())

    want = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = float((d.double() * move).sum())
    # Third derivatives times 1e-10, and the gradient's own bound.
    assert abs(got - want) <= float((grads(logits, tokens, t, dl, dn)[1] * move.abs()).sum()) + 1e-6 * (1 + abs(want))


def test_subsets_streams_and_graphs(spec):
    logits, gen = make(40, 9000, BF)
    tokens = torch.randint(0, 9000, (40,), generator=gen, device="cuda", dtype=torch.int32)
    logprob, entropy, lse, (ids, values) = run(spec, logits, tokens, None, 5)
    e2, l2 = torch.empty_like(entropy), torch.empty_like(lse)
    spec.logprobs(logits, None, None, entropy=e2)
    spec.logprobs(logits, None, None, lse=l2)
    assert torch.equal(e2, entropy) and torch.equal(l2, lse)
    i2, v2 = torch.empty_like(ids), torch.empty_like(values)
    spec.logprobs(logits, None, None, top=(i2, v2))
    assert torch.equal(i2, ids) and torch.equal(v2, values)
    lp, d = torch.zeros_like(logprob), torch.zeros_like(logits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spec.logprobs(logits, tokens, lp, lse=l2, top=(i2, v2))
        spec.logprobs_backward(logits, tokens, l2, lp, d)
    want = torch.empty_like(d)
    spec.logprobs_backward(logits, tokens, lse, logprob, want)
    for _ in range(2):
        lp.zero_(), l2.zero_(), i2.zero_(), d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lp, logprob) and torch.equal(i2, ids) and torch.equal(d, want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on_side = run(spec, logits, tokens, None, 5)
    side.synchronize()
    assert torch.equal(on_side[0], logprob) and torch.equal(on_side[3][0], ids)
    spec.logprobs(logits[:0], tokens[:0], lp[:0])  # no rows: nothing
