"""A round judged on a stream of its own, with inputs that torch's current stream is still about to write and answers that are read there at once."""
import importlib

import pytest

from test_gpu_accept import rule

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# (A round's metadata lie on the pool's stream; a call on another one first waits for the whole device, which a capture cannot.)
@pytest.mark.parametrize("pools_own,captured", [(False, False), (True, False), (True, True)])
def test_inputs_and_answers_are_waited_for(pools_own, captured):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    importlib.import_module("glm53f-afd_b200").ffi.load()
    K, marks, verify = (importlib.import_module("glm53f-afd_b200." + n) for n in ("kernel", "marks", "verify"))
    windows, vocab = [5, 2], 777
    rows = sum(windows)
    gen = torch.Generator().manual_seed(4)
    target, u = torch.randn(rows, vocab, generator=gen), torch.rand(rows, generator=gen)
    tokens = torch.zeros(rows, dtype=torch.int32)
    tokens[1:] = target.argmax(-1)[:-1].int()
    tokens[3] = (int(tokens[3]) + 1) % vocab
    greedy = torch.zeros(2)
    want = rule(windows, tokens, target, u, False, None, greedy)
    own = K.Stream(torch.cuda.Stream())
    pool = marks.KvPool(marks.KvConfig(marks.KvLayout.new(1, 0), 2, 2), own if pools_own else None)
    vf = verify.KdaVerify(pool, [None], 8, 4)
    made = [t.cuda() for t in (tokens, target, u, greedy)]
    given = [torch.zeros_like(t) for t in made]
    keep, nxt, kept, after = (torch.full((2,), -7, dtype=torch.int32, device="cuda") for _ in range(4))
    vf.verify([(pool.slot(), n) for n in windows])

    def judge():
        torch.cuda._sleep(20_000_000)  # about 10 ms
        for a, b in zip(given, made):
            a.copy_(b)
        vf.accept(*given[:3], keep, nxt, temperature=given[3], stream=own)
        kept.copy_(keep)
        after.copy_(nxt)

    torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            judge()
        for a in given:
            a.zero_()
        graph.replay()
    else:
        judge()
    assert (kept.tolist(), after.tolist()) == want and want[0] == [3, 2]
