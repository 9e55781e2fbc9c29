"""The logits' gradient at low and high temperatures, of logits far from 0 and of rows whose mask is a type's lowest value: p has the bound that it has anywhere.

Bounds, u = 2^-24, V the vocabulary.  log p = x / T - lse with |lse| of at most L, 64 for f32 logits and 256 for bf16 ones, is off by L u for 1 / T, as much for lse's own roundings, and by what lse's sum is off,
s = u (V / 512 + 300); otherwise it is (x - max) / T - log S, three roundings of a size that |log p| + log V bounds and s.  p below 2^-126 is 0.  The entropy is what the forward pass gave: to 2 s (1 + H) and 10 u (H + log V)."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_logprobs import BF, F32, INF, NAN, U, exact, heat_of, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def spec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.spec")


def grads(logits, tokens, temperature, dl, dn):
    logp, h = exact(logits, temperature)
    h, p, heat = h[:, None], logp.exp(), heat_of(temperature, len(logits))
    l, n = ((torch.zeros(len(p), 1, dtype=torch.float64, device="cuda") if g is None else g.double()[:, None]) for g in (dl, dn))
    vocab = p.shape[1]
    named = (tokens >= 0) & (tokens < vocab)
    at = tokens.long().clamp(0, vocab - 1)[:, None]
    l = l * named[:, None]
    safe = logp.masked_fill(logp == -INF, 0.0)
    d = (-l * p - n * p * (safe + h)).scatter_add_(1, at, l) / heat
    s = U * (vocab / 512 + 300)
    size = safe.abs().clamp(max=1000) + math.log(vocab + 1)
    rel = s + U * (8 * size + 20 + (512 if logits.dtype == BF else 128))
    terms = l.abs() + n.abs() * (safe.abs().clamp(max=1000) + h)
    bound = (p * rel + 2.0 ** -126) * terms + n.abs() * p * (2 * s * (1 + h) + 16 * U * (size + h))
    bound.scatter_add_(1, at, 8 * U * l.abs())
    return d, bound / heat + 1e-37


def check(spec, logits, tokens, temperature, seed=1):
    rows, vocab = logits.shape
    gen = torch.Generator(device="cuda").manual_seed(seed)
    _, entropy, lse, _ = run(spec, logits, tokens, temperature)
    dl, dn = (torch.randn(rows, generator=gen, device="cuda") for _ in range(2))
    room = torch.empty(rows * (vocab + 1) + 3, dtype=logits.dtype, device="cuda")[3:].view(rows, vocab + 1)[:, :vocab]  # (another place on the 16 bytes)
    for a, b in ((dl, None), (None, dn), (dl, dn)):
        want, bound = grads(logits, tokens, temperature, a, b)
        step = torch.finfo(logits.dtype).eps / 2 * (want.abs() + bound)
        outs = []
        for out in (torch.full((rows, vocab), 3.0, dtype=logits.dtype, device="cuda"), room, logits.clone()):
            source = out if len(outs) == 2 else logits  # in place
            spec.logprobs_backward(source, tokens, lse, a, out, temperature=temperature, entropy=entropy if b is not None else None, dentropy=b)
            over = (out.double() - want).abs() - (bound + step)
            assert (over <= 0).all(), ((out.double() - want).abs() / (bound + step)).amax(1)
            outs.append(out)
        assert torch.equal(outs[0], outs[2])  # (the same pieces of 16 bytes)
    return outs[0]


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(9, 1), (9, 300), (9, 5000), (12, 20000), (9, 131072), (300, 9001), (700, 33000), (300, 131072), (601, 131071)])
def test_temperatures(spec, dtype, rows, vocab):
    gen = torch.Generator(device="cuda").manual_seed(2)
    logits = (2.5 * torch.randn(rows, vocab, generator=gen, device="cuda")).to(dtype)
    if vocab > 100:
        logits[:, 5::17] = -INF
    t = torch.tensor([0.0, -1.0, NAN, 1.0, 1e-30, 1e38, 1e-45, 0.01, 100.0, 1e-4, 1e-8, 0.2, 1e-6], device="cuda")
    t = t.repeat(-(-rows // len(t)))[:rows]
    best, other = logits.argmax(1).int(), torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    other[-1] = -100
    check(spec, logits, best, t)
    check(spec, logits, other, t)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [7, 3000, 70000])
def test_logits_far_from_0(spec, dtype, vocab):
    gen = torch.Generator(device="cuda").manual_seed(3)
    logits = 2.5 * torch.randn(12, vocab, generator=gen, device="cuda")
    offsets = torch.tensor([0.0, 50.0, -50.0, 70.0, -70.0, 1e3, -1e3, 1e4, -1e4, 1e6, 1e30, -1e30], device="cuda")
    logits = (logits + offsets[:, None]).to(dtype)
    tokens = torch.randint(0, vocab, (12,), generator=gen, device="cuda", dtype=torch.int32)
    check(spec, logits, tokens, None)
    check(spec, logits, tokens, torch.full((12,), 0.7, device="cuda"))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 3000, 70000])
def test_masks_of_the_lowest_value(spec, dtype, vocab):
    """A row of nothing but the lowest value is one of equal logits; beside others the lowest value is none."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    logits = (2.5 * torch.randn(6, vocab, generator=gen, device="cuda")).to(dtype)
    lowest = torch.finfo(dtype).min
    logits[0], logits[1, 1::2], logits[2, 1:], logits[3], logits[4, :-1] = lowest, lowest, lowest, torch.finfo(dtype).max, -INF
    tokens = torch.tensor([0, 2, 0, vocab - 1, vocab - 1, -1], dtype=torch.int32, device="cuda")
    d = check(spec, logits, tokens, None)
    assert (d[1, 1::2] == 0).all() and (d[4] == 0).all()
    check(spec, logits, tokens, torch.tensor([0.5, 2.0, 0.5, 0.5, 1e-3, 0.3], device="cuda"))


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3001, 40000])
def test_rows_with_nothing_and_with_what_is_no_number(spec, dtype, vocab):
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = (2.5 * torch.randn(8, vocab, generator=gen, device="cuda")).to(dtype)
    logits[0], logits[7] = -INF, -INF
    logits[1, 1::2] = -INF
    logits[2, 100], logits[3, 5], logits[4] = NAN, INF, NAN
    logits[5, :] = -INF
    logits[5, 3000] = -7.0
    tokens = torch.tensor([3, 1, 7, 5, 0, 3000, -1, -1], dtype=torch.int32, device="cuda")
    _, entropy, lse, _ = run(spec, logits, tokens)
    one = torch.ones(8, device="cuda")
    for a, b in ((one, one), (one, None), (None, one)):
        d = torch.full_like(logits, 3.0)
        spec.logprobs_backward(logits, tokens, lse, a, d, entropy=None if b is None else entropy, dentropy=b)
        assert (d[[0, 5, 7]] == 0).all()
        assert (d[1, 3::2] == 0).all() and d[1, 1] == (0 if a is None else 1)  # (the token of row 1 is a masked one)
        for r in (2, 3, 4):
            assert d[r].isnan().all()
        good = torch.tensor([1, 6], device="cuda")
        want, bound = grads(logits[good], tokens[good], None, None if a is None else a[good], None if b is None else b[good])
        step = torch.finfo(dtype).eps / 2 * (want.abs() + bound)
        assert ((d[good].double() - want).abs() <= bound + step).all()
