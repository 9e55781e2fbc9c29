"""Log probabilities of tokens and alternatives that a type's lowest value masks: that value's own, as long as f32 holds it."""
import importlib
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_logprobs import BF, F32, U, exact, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def spec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    return importlib.import_module("glm53f-afd_b200.spec")


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("vocab", [40, 3000, 70000])
@pytest.mark.parametrize("rows", [4, 400])
def test_masked_tokens_and_alternatives(spec, dtype, vocab, rows):
    gen = torch.Generator(device="cuda").manual_seed(6)
    logits = (2.5 * torch.randn(rows, vocab, generator=gen, device="cuda")).to(dtype)
    lowest = torch.finfo(dtype).min
    logits[:, 3:] = lowest  # three are left
    logits[2], logits[3] = lowest, -math.inf
    logits[3, 7] = lowest
    tokens = torch.randint(3, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[0], tokens[3] = 1, 7
    for t in (None, torch.ones(rows, device="cuda"), torch.full((rows,), 2.0, device="cuda"), torch.full((rows,), 0.7, device="cuda")):
        logprob, _, _, (ids, values) = run(spec, logits, tokens, t, 8)
        logp, _ = exact(logits, t)
        for got, want in ((logprob, logp.gather(1, tokens.long()[:, None])[:, 0]), (values, torch.where(ids < 0, -math.inf, logp.gather(1, ids.long().clamp(min=0))))):
            gone = want < -3.4028235e38  # beyond f32: -inf
            assert (got[gone] == -math.inf).all()
            # A subtraction, a division and the sum's logarithm, a rounding each, and what the sum is off by.
            bound = 4 * U * want.abs() + U * (vocab / 512 + 300) + 10 * U * math.log(vocab)
            assert ((got.double() - want).abs() <= bound)[~gone].all()
        assert (values[3, 1:] == -math.inf).all() and (ids[3, 1:] == -1).all() and values[3, 0] == 0
        assert torch.equal(ids[2], torch.arange(8, dtype=torch.int32, device="cuda"))
